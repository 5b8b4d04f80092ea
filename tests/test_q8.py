"""The 8-bit cache's refusals, host arithmetic and reference, without a GPU."""
from __future__ import annotations

import copy
import ctypes
import pickle

import pytest

torch = pytest.importorskip("torch")

from jacq_amd import kivi, q8  # noqa: E402
from tests import q8_ref as ref  # noqa: E402

EINVAL, ENOMEM = 1, 3
GOOD = dict(num_heads=8, num_kv_heads=2, head_dim=64, page_size=32, max_pages_per_seq=4,
            num_pages=16)


def error(rc, code, text):
    assert rc == code and text in q8.last_error(), (rc, q8.last_error())


def test_version_and_exports():
    assert q8.lib().jacq_q8_version() == 1


@pytest.mark.parametrize("change,text", [
    (dict(num_heads=9), "multiple"), (dict(num_kv_heads=0), "multiple"),
    (dict(num_heads=34), "<= 16"), (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"),
    (dict(page_size=128), "page_size"), (dict(max_pages_per_seq=0), "max_pages"),
    (dict(max_pages_per_seq=16385), "max_pages"), (dict(num_pages=0), "num_pages"),
    (dict(codes="int4"), "codes")])
def test_geometry_refusals(change, text):
    with pytest.raises(kivi.KiviCheckError, match=text):
        q8.Q8Geometry(**{**GOOD, **change}).check()
    q8.Q8Geometry(**GOOD).check()


def test_geometry_record_is_no_attribute():
    g = q8.Q8Geometry(**GOOD)
    g.check()
    assert pickle.loads(pickle.dumps(g)) == g == copy.copy(g)
    assert "_ref" not in vars(g)
    assert g.max_seq_len() == q8.lib().jacq_q8_max_seq_len(g.ref) == 128
    assert g.page_bytes() == 2 * (2 * 32 * 64 + 8)


class Record:
    """Aligned host addresses that no call may reach: every call here is refused before it
    launches anything."""

    def __init__(self, **geo):
        self.geo = q8.Q8Geometry(**{**GOOD, **geo})
        self.pool = q8._Pool(*[4096 * (i + 1) for i in range(6)])
        self.args = q8._AttendArgs(0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0, 0, 8 * 64, 0, 0,
                                   2, 10, 5, 0, 0, 0.125, 1.0)

    def attend(self, ws=0, ws_bytes=0, pool=None, **kw):
        for k, v in kw.items():
            setattr(self.args, k, v)
        return q8.lib().jacq_q8_attend(self.geo.ref, ctypes.byref(pool or self.pool),
                                       bytes(self.args), ws, ws_bytes, None)


@pytest.mark.parametrize("kw,text", [
    (dict(batch=-1), "batch"), (dict(batch=65536), "batch"), (dict(q_dtype=2), "fp16 or bf16"),
    (dict(o_dtype=1), "queries' type"), (dict(total_q=-1), "negative"),
    (dict(CU_Q=0), "one query"), (dict(window=-1), "negative"), (dict(sinks=-1), "negative"),
    (dict(scale=float("nan")), "finite"), (dict(scale=-0.5), "positive"), (dict(decay=-0.5), "finite"),
    (dict(WEIGHTS=0x60000, max_q=65, total_q=200), "64 queries"), (dict(q_stride=500), "stride"),
    (dict(q_stride=516), "stride"), (dict(Q=0), "null"), (dict(O=0), "null"),
    (dict(SEQ_LENS=0), "null"), (dict(Q=0x10008), "16-byte"), (dict(LSE=0x60002), "4-byte")])
def test_attend_refusals(kw, text):
    error(Record().attend(**kw), EINVAL, text)


def test_attend_refuses_a_small_workspace():
    r = Record(max_pages_per_seq=1024)
    need = q8.lib().jacq_q8_attend_workspace_size(r.geo.ref, 2, 10, 5, 0)
    assert need > 0
    error(r.attend(), ENOMEM, str(need))
    error(r.attend(ws=0x100000, ws_bytes=need - 1), ENOMEM, str(need))
    error(r.attend(ws=0x100008, ws_bytes=need), EINVAL, "16-byte")


def test_pool_refusals():
    r = Record()
    for i in range(6):
        p = [4096 * (j + 1) for j in range(6)]
        p[i] = 0
        error(r.attend(pool=q8._Pool(*p)), EINVAL, "null")
        p[i] = 4096 * (i + 1) + (2 if i in (1, 3) else 8)
        error(r.attend(pool=q8._Pool(*p)), EINVAL, "aligned")


def test_packed_arguments_are_the_record():
    values = (1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 0.5, 0.25)
    assert q8._ATTEND.pack(*values) == bytes(q8._AttendArgs(*values))


def test_nothing_to_do_is_no_error():
    r = Record()
    assert r.attend(batch=0, total_q=0, CU_Q=0, max_q=0) == 0
    assert Record().attend(total_q=0, Q=0, O=0) == 0


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), "fp16 or bf16"), (dict(total=-1), "negative"), (dict(cu=0), "one new token"),
    (dict(ks=100), "NEW_K row stride"), (dict(vs=132), "NEW_V row stride"), (dict(k=0), "null"),
    (dict(v=0x20004), "16-byte"), (dict(start=0), "null"), (dict(batch=70000), "batch")])
def test_append_refusals(kw, text):
    a = dict(k=0x10000, v=0x20000, dtype=0, ks=128, vs=128, cu=0x30000, start=0x40000,
             tables=0x50000, total=7, most=7, batch=2)
    a.update(kw)
    r = Record()
    rc = q8.lib().jacq_q8_append(r.geo.ref, ctypes.byref(r.pool), a["k"], a["v"], a["dtype"],
                                 a["ks"], a["vs"], a["cu"], a["start"], a["tables"], a["total"],
                                 a["most"], a["batch"], None)
    error(rc, EINVAL, text)


@pytest.mark.parametrize("keep,sink,recent", [(-1, 0, 0), (3, 2, 2), (5, -1, 2), (5, 2, -1),
                                              (2 ** 31 - 1, 2 ** 31 - 1, 1)])
def test_evict_refusals(keep, sink, recent):
    r = Record()
    rc = q8.lib().jacq_q8_evict(r.geo.ref, *[4096] * 3, 2, keep, sink, recent, *[4096] * 4, None)
    error(rc, EINVAL, "keep")
    rc = q8.lib().jacq_q8_evict(r.geo.ref, 4096, 0, 4096, 2, 5, 1, 1, *[4096] * 4, None)
    error(rc, EINVAL, "null")


def test_read_refusals():
    r = Record()

    def read(k=0x10000, dtype=0, total=5, batch=2):
        return q8.lib().jacq_q8_read(r.geo.ref, ctypes.byref(r.pool), 4096, 4096, 4096, batch,
                                     total, k, 0x20000, dtype, None)

    error(read(dtype=3), EINVAL, "fp32")
    error(read(total=-1), EINVAL, "negative")
    error(read(k=0), EINVAL, "null")
    error(read(k=0x10008), EINVAL, "16-byte")
    assert read(total=0) == 0


# ---- the Python layer's checks, on CPU tensors: the last one refuses the device ----

@pytest.fixture
def cache():
    return q8.PagedQ8Cache(q8.Q8Geometry(**GOOD), 3, device="cpu")


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_cache_tensors(cache):
    t = dict(zip(q8.POOL, cache.pool()))
    assert q8.PagedQ8Cache.from_tensors(cache.geo, t).batch == 3
    assert cache.sequence_view(1).batch == 1
    for name in q8.POOL:
        for bad in (t[name][:, :1], t[name].to(torch.float64)):
            with pytest.raises(kivi.KiviCheckError, match=name):
                q8.PagedQ8Cache.from_tensors(cache.geo, {**t, name: bad})


def test_python_refusals(cache):
    q = torch.zeros(3, 8, 64, dtype=torch.float16)
    kv = torch.zeros(3, 2, 64, dtype=torch.float16)
    lens, tables, w = i32(3), i32(3, 4), torch.zeros(3, 4)

    def no(text, f, *a, **kw):
        with pytest.raises(kivi.KiviCheckError, match=text):
            f(*a, **kw)

    no("GPU device", cache.decode, q, lens, tables)
    no("Q must", cache.decode, q[:2], lens, tables)
    no("Q must", cache.decode, q[:, :7], lens, tables)
    no("fp16 or bf16", cache.decode, q.float(), lens, tables)
    no("side by side", cache.decode, q.transpose(0, 2).contiguous().transpose(0, 2), lens, tables)
    no("SEQ_LENS", cache.decode, q, lens.long(), tables)
    no("BLOCK_TABLES", cache.decode, q, lens, tables[:, :3])
    no("WINDOW", cache.decode, q, lens, tables, window=0)
    no("SINKS", cache.decode, q, lens, tables, sinks=-1)
    no("SCALE", cache.decode, q, lens, tables, scale=float("inf"))
    no("SCALE", cache.decode, q, lens, tables, scale=0.0)
    no("DECAY", cache.decode, q, lens, tables, weights=w, decay=-1.0)
    no("WEIGHTS", cache.decode, q, lens, tables, weights=w.double())
    no("O must", cache.decode, q, lens, tables, out=q.to(torch.bfloat16))
    no("LSE", cache.decode, q, lens, tables, lse=torch.zeros(3, 8, dtype=torch.float64))
    no("CU_Q", cache.prefill, q, i32(3), 3, lens, tables)
    no("at most 64", cache.prefill, q, i32(4), 65, lens, tables, weights=w)
    no("MAX_Q", cache.prefill, q, i32(4), -1, lens, tables)
    no("one new token", cache.append, kv[:2], kv[:2], tables, lens)
    no("NEW_V", cache.append, kv, kv.bfloat16(), tables, lens)
    no("CU_NEW", cache.append, kv, kv, tables, lens, cu_new=i32(3))
    no("START_LENS", cache.append, kv, kv, tables, i32(2))
    no("after the one before", cache.append, kv[:1].expand(3, 2, 64), kv, tables, lens)
    no("read as", cache.read, lens, lens, tables, 5, dtype=torch.int8)
    no("KEEP", cache.evict, w, lens, tables, 3, sink_pages=2, recent_pages=2)
    no("EVICTED|dim", cache.evict, w, lens, tables, 3, out=(tables, lens, w, i32(2)))
    no("GPU device", cache.evict, w, lens, tables, 3)


def test_workspace_size_of_refused_geometry_is_zero():
    g = q8._Geometry(8, 3, 64, 32, 4, 4, 0)
    assert q8.lib().jacq_q8_attend_workspace_size(ctypes.byref(g), 1, 1, 1, 0) == 0


# ---- the reference itself ----

def test_reference_codes_are_the_types_own():
    y = torch.linspace(-448, 448, 200001, dtype=torch.float64).float().double()
    assert torch.equal(ref.e4m3(y), y.float().to(torch.float8_e4m3fn).double())
    small = (torch.arange(-40, 41, dtype=torch.float64) / 2048)
    assert torch.equal(ref.e4m3(small), small.float().to(torch.float8_e4m3fn).double())


def test_a_corrected_product_sees_every_tie():
    """The writer's quotient n (1 / a), corrected once by its residual, in fp32, rounds every
    half code the way the exact quotient does: all 11-bit magnitudes against some largest ones."""
    import numpy as np
    f = np.float32
    for a in list(range(1024, 2048, 37)) + [1024, 1270, 2032, 2047]:
        inv = f(1) / f(a)
        for e in range(0, 9):
            x = np.arange(1024, 2048, dtype=np.float64) / 2 ** e
            x = x[x <= a]
            n = x * 127
            q = (n.astype(f) * inv).astype(f)
            rem = n - q.astype(np.float64) * a           # exact in 64 bits, as in the fma
            got = (q.astype(np.float64) + rem.astype(f).astype(np.float64) * inv).astype(f)
            assert np.array_equal(np.rint(got), np.rint(n / a)), (a, e)


def test_evict_reference():
    w = torch.tensor([[3.0, 1.0, 1.0, 5.0, 2.0, 9.0]])
    t = torch.tensor([[10, 11, 12, 13, 14, 15]], dtype=torch.int32)
    tables, lens, weights, gone = ref.evict(w, [5 * 16 + 3], t, 16, 3, 0, 1)
    assert tables.tolist() == [[10, 13, 14, 11, 12, 15]] and lens.tolist() == [3 * 16 + 3]
    assert weights.tolist() == [[3.0, 5.0, 2.0, 9.0, 0.0, 0.0]] and gone.tolist() == [2]
