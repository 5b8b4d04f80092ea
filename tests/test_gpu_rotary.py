"""Rotary positions on the GPU against their definition in 80 bits, and the way from a projection
through the int4 cache and back."""
from __future__ import annotations

import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import kivi_attend_ref as ref  # noqa: E402
from tests.test_gpu_kivi_attend import check, ints, offsets, randn  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rotary():
    from jacq_amd import rotary as m
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    m.lib()
    return m


def turned(rot, x, positions, inverse=False):
    """x [tokens, heads, HD] rotated, and sum(|inputs|) of each output, in 80 bits."""
    x = x.cpu().float().numpy().astype(np.longdouble)
    pos = positions.cpu().numpy().astype(np.longdouble)[:, None] * (-1 if inverse else 1)
    angle = pos * np.array(rot.speeds, dtype=np.longdouble)
    amp = np.longdouble(rot.amplitude)
    c, s = np.cos(angle)[:, None] * amp, np.sin(angle)[:, None] * amp
    out, size, rd = x.copy(), np.abs(x), rot.rotary_dim
    at = ((slice(0, rd // 2), slice(rd // 2, rd)) if rot.layout == "half" else
          (slice(0, rd, 2), slice(1, rd, 2)))
    a, b = (x[..., i] for i in at)
    out[..., at[0]], out[..., at[1]] = a * c - b * s, b * c + a * s
    for i in at:
        size[..., i] = (np.abs(a) + np.abs(b)) * amp
    return out, size


def assert_turned(rot, got, x, positions, inverse=False):
    want, size = turned(rot, x, positions, inverse)
    # the output's rounding, below fp16's normal numbers 2^-25 at most; cos and sin's 2^-22, and three
    # roundings in 32 bits
    step = ref.HALF_STEP[got.dtype]
    tol = step * np.abs(want) + size * (1 + step) * (2.0 ** -22 + 3 * 2.0 ** -24)
    tol += 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -149
    err = np.abs(got.cpu().double().numpy().astype(np.longdouble) - want)
    assert (err <= tol).all(), float((err / tol).max())
    rd = rot.rotary_dim
    assert torch.equal(got[..., rd:], x[..., rd:].to(got.dtype))  # what does not turn is copied


DTYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,rd", [(64, 64), (128, 128), (128, 32), (64, 16), (80, 20), (128, 2),
                                   (96, 72), (256, 256), (10, 6)])
def test_rotation(rotary, layout, dtype, hd, rd):
    gen = torch.Generator("cuda").manual_seed(hd + rd)
    rot = rotary.Rotary(hd, rd, base=500000.0, layout=layout)
    for tokens, heads, kv in ((1, 1, 1), (3, 5, 2), (70, 7, 0), (260, 24, 3)):
        q = randn(gen, tokens, heads, hd, dtype=dtype)
        k = randn(gen, tokens, kv, hd, dtype=dtype) if kv else None
        pos = torch.randint(-5, 1 << 20, (tokens,), generator=gen, device="cuda",
                            dtype=random.Random(tokens).choice([torch.int32, torch.int64]))
        qo, ko = rot.rotate(q, k, pos)
        assert qo.dtype == dtype and (ko is None) == (k is None)
        assert_turned(rot, qo, q, pos)
        if kv:
            assert_turned(rot, ko, k, pos)
    for kind, extra in (("linear", {}), ("base", {}), ("turns", {"length": 8192}),
                        ("turns", {"amplitude": 0.5})):
        scaled = rotary.Rotary(hd, rd, layout=layout, scaling=rotary.Scaling(kind, 4.0, **extra))
        assert_turned(scaled, scaled.rotate(q, k, pos)[0], q, pos)


def test_far_positions_lose_nothing(rotary):
    gen = torch.Generator("cuda").manual_seed(5)
    rot = rotary.Rotary(128)
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 12345, -2 ** 45 + 7, 999983],
                       device="cuda")
    q = randn(gen, 8, 3, 128, dtype=torch.float32)
    # 2^45 positions of 64-bit speeds: the reference's 80 bits hold an angle of 2^45 to 2^-19
    got, _ = rot.rotate(q, None, pos)
    near = pos.abs() < 2 ** 32
    assert_turned(rot, got[near], q[near], pos[near])
    # far ones by whole numbers: the fraction of a turn as an integer product
    for i in torch.nonzero(~near)[:, 0].tolist():
        turns = [int(pos[i]) * t % 2 ** 64 for t in rot._turns]
        angle = np.array(turns, dtype=np.longdouble) / np.longdouble(2) ** 63 * np.longdouble(np.pi)
        a, b = q[i, :, :64].cpu().numpy(), q[i, :, 64:].cpu().numpy()
        want = np.concatenate((a * np.cos(angle) - b * np.sin(angle),
                               b * np.cos(angle) + a * np.sin(angle)), -1)
        assert np.abs(got[i].cpu().numpy() - want).max() < 8 * 2.0 ** -22


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_a_projection_outputs_in_place_and_of_other_types(rotary, dtype):
    gen = torch.Generator("cuda").manual_seed(9)
    nh, nkv, hd, tokens = 6, 2, 64, 37
    for layout in ("half", "interleaved"):
        rot = rotary.Rotary(hd, 32, layout=layout)
        for lead in (0, 8, 3):  # 3: rows that allow no wide load
            qkv = randn(gen, tokens, lead + (nh + 2 * nkv) * hd, dtype=dtype)
            before = qkv.clone()
            pos = torch.arange(100, 100 + tokens, device="cuda", dtype=torch.int32)
            q = qkv[:, lead:lead + nh * hd].unflatten(1, (nh, hd))
            k = qkv[:, lead + nh * hd:lead + (nh + nkv) * hd].unflatten(1, (nkv, hd))
            want = rot.rotate(q.contiguous(), k.contiguous(), pos)
            got = rot.rotate(q, k, pos)
            assert torch.equal(qkv, before)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            half, _ = rot.rotate(q, None, pos, q_out=torch.empty(tokens, nh, hd, device="cuda",
                                                                 dtype=torch.float16))
            assert_turned(rot, half, q, pos)
            as_half = rot.rotate(q, k, pos, k_dtype=torch.float16)[1]
            assert as_half.dtype == torch.float16
            assert_turned(rot, as_half, k, pos)
            # into its own place: the rest of the projection stays
            rot.rotate(q, k, pos, q_out=q, k_out=k)
            assert torch.equal(q, want[0]) and torch.equal(k, want[1])
            rest = torch.cat((before[:, :lead], before[:, lead + (nh + nkv) * hd:]), 1)
            assert torch.equal(torch.cat((qkv[:, :lead], qkv[:, lead + (nh + nkv) * hd:]), 1), rest)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_the_inverse_is_the_gradient_and_the_way_back(rotary, layout):
    gen = torch.Generator("cuda").manual_seed(2)
    rot = rotary.Rotary(64, 48, layout=layout, scaling=rotary.Scaling("turns", 4.0, length=512))
    pos = torch.randint(0, 5000, (9,), generator=gen, device="cuda")
    x, g, d = (randn(gen, 9, 4, 64, dtype=torch.float32) for _ in range(3))
    back, _ = rot.rotate(g, None, pos, inverse=True)
    assert_turned(rot, back, g, pos, inverse=True)
    # the rotation is linear: <g, R(x + d) - R(x)> = <R^T g, d>
    f = [turned(rot, t, pos)[0] for t in (x + d, x)]
    slope = float((g.cpu().double().numpy() * (f[0] - f[1])).sum())
    # sums of 2304 products of sizes up to about 20, each within 2^-20 of itself
    assert abs(slope - float((back.double() * d.double()).sum())) < 2304 * 20 * 2.0 ** -20
    plain = rotary.Rotary(64, layout=layout)
    there, _ = plain.rotate(x, None, pos)
    again, _ = plain.rotate(there, None, pos, inverse=True)
    assert float((again - x).abs().max()) < 16 * 2.0 ** -21  # two rotations of values up to 5


def test_not_finite_values_stay_in_their_pair(rotary):
    rot = rotary.Rotary(64, 32)
    x = torch.ones(4, 2, 64, device="cuda")
    x[1, 0, 3], x[2, 1, 40] = float("nan"), float("inf")
    got, _ = rot.rotate(x, None, torch.arange(4, device="cuda"))
    bad = ~got.isfinite()
    want = torch.zeros_like(bad)
    want[1, 0, 3] = want[1, 0, 19] = want[2, 1, 40] = True
    assert torch.equal(bad, want)


def test_captured_and_replayed_with_new_positions(rotary):
    gen = torch.Generator("cuda").manual_seed(3)
    rot = rotary.Rotary(128)
    q, k = randn(gen, 40, 8, 128), randn(gen, 40, 2, 128)
    pos = torch.zeros(40, dtype=torch.int32, device="cuda")
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    rot.rotate(q, k, pos, q_out=qo, k_out=ko)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rot.rotate(q, k, pos, q_out=qo, k_out=ko)
    for i in range(4):
        pos.copy_(torch.arange(i * 1000, i * 1000 + 40))
        want = rot.rotate(q, k, pos)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_prompt_then_tokens_through_the_int4_cache(rotary, dtype):
    """What a program does of a layer: rotate, append, attend; and reads back what it wrote."""
    from jacq_amd import kivi
    gen = torch.Generator("cuda").manual_seed(7)
    nh, nkv, hd, residual, n = 10, 2, 128, 64, 190
    geo = kivi.KiviGeometry(nh, nkv, hd, 16, 32, residual, 16, 40)
    cache = kivi.PagedKiviCache(geo, 2)
    tables = torch.randperm(40, generator=gen, device="cuda")[:32].to(torch.int32).view(2, 16)
    rot = rotary.Rotary(hd, layout="half")
    lens = [0, 0]
    for m in (n, 1, 3, 1):
        qkv = randn(gen, 2 * m, (nh + 2 * nkv) * hd, dtype=dtype)
        pos = torch.cat([torch.arange(x, x + m) for x in lens]).to("cuda", torch.int32)
        q, k, v = (x.unflatten(1, (-1, hd)) for x in qkv.split([nh * hd, nkv * hd, nkv * hd], 1))
        q, k = rot.rotate(q, k, pos, k_dtype=torch.float16)
        start = ints(*lens)
        cache.append(k.view(2, m, nkv, hd), v.half().contiguous().view(2, m, nkv, hd), tables, start)
        lens = [x + m for x in lens]
        cu = offsets([m, m])
        o = cache.prefill(q, ints(*cu), m, ints(*lens), tables)
        check(cache, tables, lens, q, cu, o)
        if m == 1 and dtype == torch.float16:  # the int4 cache's own decode is of the same cache
            d = cache.decode(q, ints(*lens), tables)
            assert float((d - o.float()).abs().max()) < 4e-3  # its bound and as much again
    got = cache.read(ints(0, 0), ints(*lens), tables, sum(lens))
    for b in range(2):
        want = ref.exact_values(cache, tables, b, lens[b])[:2]
        for x, y in zip(got, want):
            assert torch.equal(x[b * lens[0]:(b + 1) * lens[0]], ref.to_half(y.transpose(0, 1)))
