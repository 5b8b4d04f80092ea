"""Rotary positions of queries and keys (include/jacq_rotary.h): what new tokens go
through before ``jacq_amd.kivi`` or ``jacq_amd.q8`` appends them and attends with them.

    rot = Rotary(128, base=500000.0, scaling=Scaling("turns", 8.0, length=8192))
    q, k = rot.rotate(q, k, positions)         # slices of a fused projection, one launch
    cache.append(k[:, None], v[:, None], tables, start_lens)
    o = cache.prefill(q, None, 1, start_lens + 1, tables)

The angles are exact at any position: a frequency is a 64-bit fraction of a turn, and so
is its product with a position.  The object holds no device memory; a call can be
captured and replayed with new positions.  It has no counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass
from fractions import Fraction

import torch

from jacq_amd import kivi as _kivi
from jacq_amd.kivi import DTYPES, FLOAT_MAX, KiviLaunchError, _check, check_shape

LAYOUTS = {"half": 0, "interleaved": 1}
MAX_DIM = 256  # channels of a head that turn
_SCALINGS = ("linear", "base", "turns")
_ARGS = struct.Struct("@6P4q11if")

_lib: ctypes.CDLL | None = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        L = _kivi.lib()
        L.jacq_rotary_last_error.restype = ctypes.c_char_p
        L.jacq_rotary.argtypes = [ctypes.c_void_p, ctypes.c_void_p]  # the record: packed bytes
        L.jacq_rotary.restype = ctypes.c_int
        _lib = L
    return _lib


@dataclass(frozen=True)
class Scaling:
    """How frequencies are slowed for contexts ``factor`` times longer than a model learned.

    linear   every frequency by the factor
    base     a larger base: the slowest frequency by the factor, the fastest not at all
    turns    by how often a pair turns over ``length`` tokens (what the model learned):
             frequencies of at most ``slow`` turns by the factor, of ``fast`` and more not at
             all, in between a mean of both that is linear in the turns; cosines and sines
             times ``amplitude`` (by default 0.1 ln(factor) + 1)

    A model whose mean of both is linear in the pair's index, or another one, gives its frequencies
    to ``Rotary`` as ``speeds``."""
    kind: str
    factor: float
    length: int = 4096
    slow: float = 1.0
    fast: float = 32.0
    amplitude: float | None = None

    def check(self) -> None:
        _check(self.kind in _SCALINGS, "scaling must be one of ", _SCALINGS, ", got ", self.kind)
        _check(1.0 <= self.factor < math.inf, "a scaling's factor must be at least 1 and finite")
        _check(self.length >= 1 and 0.0 <= self.slow < self.fast < math.inf,
               "a scaling's length must be positive, and 0 <= SLOW < FAST, finite")
        _check(self.amplitude is None or 0.0 < self.amplitude < math.inf,
               "a scaling's amplitude must be positive and finite")


def frequencies(rotary_dim: int, base: float = 10000.0, scaling: Scaling | None = None):
    """Radians a position of each pair, and the amplitude of cosine and sine."""
    if scaling is not None and scaling.kind == "base":
        try:
            base *= scaling.factor ** (rotary_dim / max(1, rotary_dim - 2))
        except OverflowError:
            base = math.inf
        _check(base < math.inf, "the scaled base must be finite")
    f = [base ** (-2 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling is None or scaling.kind == "base":
        return f, 1.0
    if scaling.kind == "linear":
        return [x / scaling.factor for x in f], 1.0
    out = []
    for x in f:
        turns = scaling.length * x / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - scaling.slow) / (scaling.fast - scaling.slow)))
        out.append(x * (keep + (1.0 - keep) / scaling.factor))
    amplitude = scaling.amplitude
    return out, 0.1 * math.log(scaling.factor) + 1.0 if amplitude is None else amplitude


# 2 pi to 2^-128, so that a frequency's 64 bits are its own: 106 bits are two doubles
_TWO_PI = (2 * (Fraction(3.141592653589793) + Fraction(1.2246467991473532e-16))).as_integer_ratio()


def _turns(f: float) -> int:
    """f radians in 2^-64 turns, to the nearest, ties to even.  In whole numbers: fractions, which look for
    common divisors, took 10 us."""
    num, den = f.as_integer_ratio()
    num, den = num * _TWO_PI[1] << 64, den * _TWO_PI[0]
    turns, rest = divmod(num, den)
    return (turns + (2 * rest > den or (2 * rest == den and turns & 1))) % (1 << 64)


class Rotary:
    """The rotation of one model's heads: the first ``rotary_dim`` channels (all by default), in
    pairs i, i + rotary_dim / 2 (layout "half") or 2 i, 2 i + 1 ("interleaved"), pair i by base **
    (-2 i / rotary_dim) radians a position, scaled as ``scaling`` says; or by ``speeds``, the radians
    a position of each pair, with ``amplitude``."""

    def __init__(self, head_dim: int, rotary_dim: int | None = None, base: float = 10000.0,
                 layout: str = "half", scaling: Scaling | None = None, speeds=None,
                 amplitude: float | None = None):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        _check(2 <= head_dim <= 1024 and head_dim % 2 == 0,
               "head_dim must be even and in [2, 1024], got ", head_dim)
        _check(2 <= rotary_dim <= min(head_dim, MAX_DIM) and rotary_dim % 2 == 0,
               "rotary_dim must be even, in [2, ", MAX_DIM, "] and at most head_dim, got ", rotary_dim)
        _check(layout in LAYOUTS, "layout must be one of ", tuple(LAYOUTS), ", got ", layout)
        if scaling is not None:
            scaling.check()
        if speeds is None:
            _check(1.0 <= base < math.inf, "base must be at least 1 and finite, got ", base)
            speeds, own = frequencies(rotary_dim, base, scaling)
        else:
            _check(scaling is None, "scaling is for the base's frequencies, not for given speeds")
            speeds, own = [float(x) for x in speeds], 1.0
            _check(len(speeds) == rotary_dim // 2, "speeds must be rotary_dim / 2 = ",
                   rotary_dim // 2, " numbers, got ", len(speeds))
            _check(all(math.isfinite(x) for x in speeds), "speeds must be finite")
        amplitude = own if amplitude is None else float(amplitude)
        _check(abs(amplitude) <= FLOAT_MAX, "amplitude must be finite in fp32")
        self.head_dim, self.rotary_dim, self.layout = head_dim, rotary_dim, layout
        self.speeds, self.amplitude = tuple(speeds), amplitude
        self._turns = (ctypes.c_uint64 * len(speeds))(*[_turns(x) for x in speeds])

    def __getstate__(self):  # copies and pickles make their own record
        return {n: v for n, v in vars(self).items() if n != "_turns"}

    def __setstate__(self, state: dict) -> None:
        vars(self).update(state)
        self._turns = (ctypes.c_uint64 * len(self.speeds))(*[_turns(x) for x in self.speeds])

    def _rows(self, t: torch.Tensor, tokens: int, heads: int | None, name: str) -> int:
        """Checks; the elements between token rows."""
        hd, shape = self.head_dim, t.shape
        _check(len(shape) == 3 and shape[0] == tokens and shape[2] == hd
               and (heads is None or shape[1] == heads), name, " must be [", tokens, ", ",
               "heads" if heads is None else heads, ", ", hd, "], got ", tuple(shape))
        _check(t.dtype in DTYPES, name, " must be fp16, bf16 or fp32")
        if t.is_contiguous():
            return shape[1] * hd
        _check(t.numel() == 0 or (t.stride(2) == 1 and (shape[1] == 1 or t.stride(1) == hd)), name,
               " must have its heads side by side")
        if tokens <= 1:
            return shape[1] * hd
        _check(t.numel() == 0 or t.stride(0) >= shape[1] * hd, name,
               " must have a token's row after the one before")
        return max(t.stride(0), shape[1] * hd)

    def _quick(self, t: torch.Tensor, index: int) -> int:
        """The elements between token rows, or 0 for the named checks to say what is wrong: they
        take the host longer than a small call takes the GPU."""
        shape, stride, hd = t.shape, t.stride(), self.head_dim
        return (stride[0] if len(shape) == 3 and shape[2] == hd and stride[2] == 1 and stride[1] == hd
                and stride[0] >= shape[1] * hd > 0 and t.dtype in DTYPES and t.get_device() == index
                else 0)

    def rotate(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
               inverse: bool = False, k_dtype: torch.dtype | None = None,
               q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
        """q [tokens, heads, HD] and k [tokens, kv heads, HD] of one type, whose rows may lie apart
        (slices of a fused projection), at positions [tokens] int32 or int64, of any sign -> the
        same rotated: new tensors of their type (k of k_dtype: the int4 cache takes fp16), or
        q_out, k_out, of any type, which may be q and k themselves and must overlap neither
        otherwise.  k may be None.  inverse: by the negative angles; with an amplitude of 1 the
        way back, with any the gradient of this rotation for the gradient of its outputs, which
        carry no autograd graph themselves."""
        shape, dtype, index = q.shape, q.dtype, q.get_device()
        tokens = shape[0] if len(shape) else 0
        q_stride, k_stride = self._quick(q, index), 0
        fits = (q_stride and index >= 0 and positions.shape == (tokens,)
                and (positions.dtype is torch.int32 or positions.dtype is torch.int64)
                and positions.is_contiguous() and positions.get_device() == index)
        if k is not None:
            k_stride = self._quick(k, index)
            fits = fits and k_stride and k.shape[0] == tokens and k.dtype is dtype
        fits = fits and q_out is None and k_out is None and (k_dtype is None or k is not None)
        if not fits:
            q_stride = self._rows(q, tokens, None, "Q")
            if k is not None:
                k_stride = self._rows(k, tokens, None, "K")
                _check(k.dtype == dtype, "K must be of Q's type")
            else:
                _check(k_out is None and k_dtype is None, "K_OUT and K_DTYPE are for K")
            check_shape(positions, (tokens,), "POSITIONS")
            _check(positions.dtype in (torch.int32, torch.int64) and positions.is_contiguous(),
                   "POSITIONS must be contiguous int32 or int64")
        heads, kv_heads = shape[1], 0 if k is None else k.shape[1]
        _check(k_dtype is None or k_dtype in DTYPES, "K_DTYPE must be fp16, bf16 or fp32")
        strides = [q_stride, k_stride, heads * self.head_dim, kv_heads * self.head_dim]
        if q_out is None:  # empty_like is the quicker one, where it gives rows side by side
            q_out = (torch.empty_like(q) if fits else
                     torch.empty((tokens, heads, self.head_dim), dtype=dtype, device=q.device))
        else:
            strides[2] = self._rows(q_out, tokens, heads, "Q_OUT")
        if k is not None:
            if k_out is None:
                k_out = (torch.empty_like(k, dtype=k_dtype or dtype) if fits else
                         torch.empty((tokens, kv_heads, self.head_dim), dtype=k_dtype or dtype,
                                     device=q.device))
            else:
                strides[3] = self._rows(k_out, tokens, kv_heads, "K_OUT")
                _check(k_dtype is None or k_out.dtype == k_dtype, "K_OUT must be of K_DTYPE")
        if not fits:
            _check(index >= 0, "Q must be on a GPU device, got ", q.device)
            for t, name in ((k, "K"), (positions, "POSITIONS"), (q_out, "Q_OUT"), (k_out, "K_OUT")):
                _check(t is None or t.get_device() == index, name, " must be on Q's device")
            for t, out, i, name in ((q, q_out, 0, "Q_OUT"), (k, k_out, 1, "K_OUT")):
                if t is not None and t.data_ptr() == out.data_ptr() and t.numel():
                    _check(t.dtype == out.dtype and strides[i] == strides[i + 2], name,
                           " at its input's place must be of its type and stride")
        args = _ARGS.pack(q.data_ptr(), 0 if k is None else k.data_ptr(), positions.data_ptr(),
                          q_out.data_ptr(), 0 if k is None else k_out.data_ptr(),
                          ctypes.addressof(self._turns), *strides, tokens, heads, kv_heads,
                          self.head_dim, self.rotary_dim, LAYOUTS[self.layout], DTYPES[dtype],
                          DTYPES[q_out.dtype], 0 if k is None else DTYPES[k_out.dtype],
                          positions.dtype == torch.int64, bool(inverse), self.amplitude)
        fn = lib().jacq_rotary
        if torch._C._cuda_getDevice() == index:
            rc = fn(args, torch._C._cuda_getCurrentRawStream(index))
        else:
            with torch.cuda.device(index):
                rc = fn(args, torch._C._cuda_getCurrentRawStream(index))
        if rc != 0:
            raise KiviLaunchError(lib().jacq_rotary_last_error().decode())
        return q_out, k_out
