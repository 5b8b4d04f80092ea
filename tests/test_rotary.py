"""Refusals and frequencies of the rotary positions, without a GPU."""
from __future__ import annotations

import copy
import math
import pickle

import pytest

torch = pytest.importorskip("torch")

from jacq_amd import kivi, rotary  # noqa: E402

EINVAL = 1
FIELDS = ("Q", "K", "POSITIONS", "Q_OUT", "K_OUT", "TURNS", "q_stride", "k_stride", "q_out_stride",
          "k_out_stride", "tokens", "num_heads", "num_kv_heads", "head_dim", "rotary_dim", "layout",
          "dtype", "q_out_dtype", "k_out_dtype", "positions64", "inverse", "amplitude")
ARGS = dict(zip(FIELDS, (0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0x60000, 512, 128, 512, 128, 5, 8,
                         2, 64, 64, 0, 0, 0, 0, 0, 0, 1.0)))


def call(**kw):
    """Host addresses that no call may reach: each is refused before it reads or launches anything."""
    return rotary.lib().jacq_rotary(rotary._ARGS.pack(*{**ARGS, **kw}.values()), None)


@pytest.mark.parametrize("kw,text", [
    (dict(tokens=-1), "negative"), (dict(num_heads=-1), "negative"), (dict(num_kv_heads=65537), "65536"),
    (dict(head_dim=63), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(head_dim=2048), "head_dim"),
    (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=31), "rotary_dim"),
    (dict(rotary_dim=66), "rotary_dim"),
    (dict(head_dim=512, rotary_dim=258, q_stride=4096, k_stride=1024, q_out_stride=4096,
          k_out_stride=1024), "rotary_dim"),
    (dict(layout=2), "layout"), (dict(dtype=3), "fp16, bf16 or fp32"), (dict(q_out_dtype=-1), "fp16"),
    (dict(k_out_dtype=5), "fp16"), (dict(amplitude=float("inf")), "amplitude"),
    (dict(amplitude=float("nan")), "amplitude"), (dict(q_stride=511), "stride"),
    (dict(k_stride=127), "stride"), (dict(q_out_stride=0), "stride"), (dict(k_out_stride=-128), "stride"),
    (dict(Q=0), "null"), (dict(K=0), "null"), (dict(POSITIONS=0), "null"), (dict(Q_OUT=0), "null"),
    (dict(K_OUT=0), "null"), (dict(TURNS=0), "null"), (dict(Q=0x10001), "aligned"),
    (dict(POSITIONS=0x30002), "aligned"), (dict(POSITIONS=0x30004, positions64=1), "aligned")])
def test_refusals(kw, text):
    rc = call(**kw)
    assert rc == EINVAL and text in rotary.lib().jacq_rotary_last_error().decode(), (
        rc, rotary.lib().jacq_rotary_last_error())


def test_calls_of_nothing_launch_nothing():
    assert call(tokens=0, Q=0, K=0, POSITIONS=0, TURNS=0) == 0
    assert call(num_heads=0, num_kv_heads=0, Q=0, K=0) == 0


@pytest.mark.parametrize("kw,text", [
    (dict(head_dim=63), "head_dim"), (dict(rotary_dim=130), "rotary_dim"), (dict(rotary_dim=5), "rotary_dim"),
    (dict(layout="both"), "layout"), (dict(base=0.5), "base"), (dict(base=math.inf), "base"),
    (dict(speeds=[1.0]), "speeds"), (dict(speeds=[math.nan] * 64), "finite"),
    (dict(speeds=[1.0] * 64, scaling=rotary.Scaling("linear", 2.0)), "speeds"),
    (dict(amplitude=math.inf), "amplitude"), (dict(scaling=rotary.Scaling("cubic", 2.0)), "scaling"),
    (dict(scaling=rotary.Scaling("linear", 0.5)), "factor"),
    (dict(scaling=rotary.Scaling("turns", 2.0, slow=4.0, fast=4.0)), "SLOW"),
    (dict(scaling=rotary.Scaling("turns", 2.0, length=0)), "length"),
    (dict(scaling=rotary.Scaling("turns", 2.0, amplitude=0.0)), "amplitude")])
def test_plans_are_checked(kw, text):
    with pytest.raises(kivi.KiviCheckError, match=text):
        rotary.Rotary(**{"head_dim": 128, **kw})


Q, K, POS = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32)


@pytest.mark.parametrize("kw,text", [
    (dict(q=Q[..., :63]), "Q must be"), (dict(q=Q.double()), "Q must be"), (dict(k=K[:2]), "K must be"),
    (dict(q=Q.transpose(0, 1).contiguous().transpose(0, 1)), "side by side"),
    (dict(q=Q[:1].expand(3, 4, 64)), "one before"), (dict(k=K.half()), "Q's type"),
    (dict(positions=POS[:2]), "POSITIONS"), (dict(positions=POS.float()), "POSITIONS"),
    (dict(positions=POS.repeat_interleave(2)[::2]), "contiguous"), (dict(k=None, k_out=K), "for K"),
    (dict(k=None, k_dtype=torch.float16), "for K"), (dict(k_dtype=torch.float64), "K_DTYPE"),
    (dict(k_out=K, k_dtype=torch.float16), "K_DTYPE"), (dict(q_out=Q[:, :3]), "Q_OUT"),
    (dict(k_out=Q), "K_OUT"), (dict(), "GPU device")])
def test_python_refusals(kw, text):
    with pytest.raises(kivi.KiviCheckError, match=text):
        rotary.Rotary(64).rotate(**{**dict(q=Q, k=K, positions=POS), **kw})


def test_frequencies():
    f, amp = rotary.frequencies(64, 10000.0)
    assert amp == 1.0 and f[0] == 1.0 and len(f) == 32
    assert all(abs(f[i] / 10000.0 ** (-i / 32) - 1) < 1e-14 for i in range(32))
    linear, _ = rotary.frequencies(64, 10000.0, rotary.Scaling("linear", 4.0))
    assert linear == [x / 4.0 for x in f]
    based, _ = rotary.frequencies(64, 10000.0, rotary.Scaling("base", 4.0))
    assert based[0] == 1.0 and abs(based[-1] * 4.0 / f[-1] - 1) < 1e-12
    s = rotary.Scaling("turns", 4.0, length=4096, slow=1.0, fast=32.0)
    turns, amp = rotary.frequencies(64, 10000.0, s)
    assert amp == 0.1 * math.log(4.0) + 1
    for x, y in zip(f, turns):
        n = 4096 * x / (2 * math.pi)
        assert y == x if n >= 32 else y == x / 4 if n <= 1 else x / 4 < y < x
    assert rotary.frequencies(2, 10000.0, rotary.Scaling("base", 4.0))[0] == [1.0]


def test_turns_are_fractions_of_2_to_the_64():
    assert rotary._turns(0.0) == 0
    # a whole turn in doubles is 2 pi less 2.4e-16: as many 2^-64 turns short of one
    short = 2 ** 64 - rotary._turns(2 * math.pi)
    assert abs(short / 2 ** 64 * 2 * math.pi - 2.4492935982947064e-16) < 2.0 ** -64
    assert rotary._turns(-0.5) == 2 ** 64 - rotary._turns(0.5)


def test_plans_can_be_copied_and_pickled():
    r = rotary.Rotary(128, 64, layout="interleaved", scaling=rotary.Scaling("turns", 8.0))
    for other in (copy.deepcopy(r), pickle.loads(pickle.dumps(r))):
        assert other.speeds == r.speeds and list(other._turns) == list(r._turns)
        assert (other.head_dim, other.rotary_dim, other.layout, other.amplitude) == (
            128, 64, "interleaved", r.amplitude)
