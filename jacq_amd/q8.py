"""The 8-bit paged KV cache (include/jacq_q8.h): one scale per block of tokens and
kv head, int8 or e4m3 codes, beside the int4 cache of ``jacq_amd.kivi``.

``PagedQ8Cache`` holds the page pool and the sequences' tails (the block in
progress, fp16) and calls the library:

    geo = Q8Geometry(40, 8, 128, page_size=32, max_pages_per_seq=512, num_pages=8192)
    cache = PagedQ8Cache(geo, batch=64)
    cache.append(k, v, tables, start_lens)                # a token per sequence
    o = cache.decode(q, seq_lens, tables)                 # one query per sequence
    o = cache.decode(q, seq_lens, tables, window=4096, sinks=4)
    o = cache.prefill(q, cu_q, max_q, seq_lens, tables)   # prompts, ragged
    o = cache.decode(q, seq_lens, tables, weights=w)      # adds up the blocks' weights
    tables, seq_lens, w, evicted = cache.evict(w, seq_lens, tables, keep=256)

There is no fallback: without libjacq_kivi.so the import of the native layer
raises ``NativeLibraryMissing``.  It has no counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass

import torch

from jacq_amd import kivi as _kivi
from jacq_amd.kivi import KiviLaunchError, _check, check_shape

CODES = {"int8": 0, "e4m3": 1}
DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
MAX_WEIGHTED_QUERIES = 64  # queries per sequence of a call that adds up block weights

_vp, _i32, _i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


class _Geometry(ctypes.Structure):
    _fields_ = [(n, _i32) for n in ("num_heads", "num_kv_heads", "head_dim", "page_size",
                                    "max_pages_per_seq", "num_pages", "codes")]


class _Pool(ctypes.Structure):
    _fields_ = [(n, _vp) for n in ("k_code", "k_scale", "v_code", "v_scale", "k_tail", "v_tail")]


# _AttendArgs packed at once: setting its fields one by one takes as long as a launch
_ATTEND = struct.Struct("@7Pq7i2f4x")


class _AttendArgs(ctypes.Structure):
    _fields_ = ([(n, _vp) for n in ("Q", "CU_Q", "SEQ_LENS", "BLOCK_TABLES", "O", "LSE",
                                    "WEIGHTS")]
                + [("q_stride", _i64)]
                + [(n, _i32) for n in ("q_dtype", "o_dtype", "batch", "total_q", "max_q", "window",
                                       "sinks")]
                + [("scale", ctypes.c_float), ("decay", ctypes.c_float)])


_lib: ctypes.CDLL | None = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    L = _kivi.lib()
    geo, pool = ctypes.POINTER(_Geometry), ctypes.POINTER(_Pool)
    L.jacq_q8_version.restype = ctypes.c_int
    L.jacq_q8_last_error.restype = ctypes.c_char_p
    L.jacq_q8_check_geometry.argtypes = [geo]
    L.jacq_q8_check_geometry.restype = ctypes.c_int
    L.jacq_q8_max_seq_len.argtypes = [geo]
    L.jacq_q8_max_seq_len.restype = _i64
    L.jacq_q8_append.argtypes = [geo, pool, _vp, _vp, _i32, _i64, _i64, _vp, _vp, _vp, _i32, _i32,
                                 _i32, _vp]
    L.jacq_q8_append.restype = ctypes.c_int
    L.jacq_q8_attend_workspace_size.argtypes = [geo, _i32, _i32, _i32, _i32]
    L.jacq_q8_attend_workspace_size.restype = ctypes.c_size_t
    L.jacq_q8_attend.argtypes = [geo, pool, _vp, _vp, ctypes.c_size_t, _vp]  # args: packed bytes
    L.jacq_q8_attend.restype = ctypes.c_int
    L.jacq_q8_read.argtypes = [geo, pool, _vp, _vp, _vp, _i32, _i32, _vp, _vp, _i32, _vp]
    L.jacq_q8_read.restype = ctypes.c_int
    L.jacq_q8_evict.argtypes = [geo, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _vp, _vp, _vp, _vp, _vp]
    L.jacq_q8_evict.restype = ctypes.c_int
    _lib = L
    return L


def last_error() -> str:
    return lib().jacq_q8_last_error().decode()


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


@dataclass(frozen=True)
class Q8Geometry(_kivi._WithRecord):
    num_heads: int
    num_kv_heads: int
    head_dim: int
    page_size: int = 32
    max_pages_per_seq: int = 128
    num_pages: int = 1
    codes: str = "int8"

    @property
    def gqa(self) -> int:
        return self.num_heads // self.num_kv_heads

    @property
    def ref(self):
        """The argument record by reference, made once: the fields never change."""
        try:
            return self._ref
        except AttributeError:
            _check(self.codes in CODES, "codes must be one of ", sorted(CODES), ", got ",
                   self.codes)
            rec = _Geometry(self.num_heads, self.num_kv_heads, self.head_dim, self.page_size,
                            self.max_pages_per_seq, self.num_pages, CODES[self.codes])
            object.__setattr__(self, "_ref", ctypes.byref(rec))
            return self._ref

    def __getstate__(self):  # copies and pickles carry the attributes, not the record
        return dict(vars(self))

    def check(self) -> None:
        if lib().jacq_q8_check_geometry(self.ref) != 0:
            raise _kivi.KiviCheckError(last_error())

    def max_seq_len(self) -> int:
        return self.max_pages_per_seq * self.page_size

    def page_bytes(self) -> int:
        """Bytes of one page, all kv heads: codes and scales of K and V."""
        return self.num_kv_heads * (2 * self.page_size * self.head_dim + 8)


POOL = ("k_code", "k_scale", "v_code", "v_scale", "k_tail", "v_tail")


class PagedQ8Cache:
    """Page pool and tails of ``batch`` sequences on one device.

    k_code  uint8 [num_pages, NKV, P, HD]   v_code  uint8 [num_pages, NKV, HD, P]
    k_scale, v_scale  fp32 [num_pages, NKV]
    k_tail, v_tail    fp16 [batch, NKV, P, HD], the seq_len % P newest tokens

    A block's value is code * scale (int8: (code - 128) * scale).  Lengths, offsets
    and block tables are int32 on the cache's device; queries and new tokens are fp16
    or bf16 whose token rows may lie apart (a slice of a fused projection), the rest
    is contiguous.  Calls run on the current stream of the cache's device; a decode
    after an append on the same stream sees it.  A workspace that is not given comes
    from torch's allocator, as the outputs do."""

    def __init__(self, geo: Q8Geometry, batch: int, device="cuda"):
        geo.check()
        g, dev = geo, torch.device(device)
        _check(batch >= 1, "batch must be positive")
        shape = (g.num_pages, g.num_kv_heads)
        self._set(geo, {
            "k_code": torch.zeros((*shape, g.page_size, g.head_dim), dtype=torch.uint8, device=dev),
            "k_scale": torch.zeros(shape, dtype=torch.float32, device=dev),
            "v_code": torch.zeros((*shape, g.head_dim, g.page_size), dtype=torch.uint8, device=dev),
            "v_scale": torch.zeros(shape, dtype=torch.float32, device=dev),
            "k_tail": torch.zeros((batch, g.num_kv_heads, g.page_size, g.head_dim),
                                  dtype=torch.float16, device=dev),
            "v_tail": torch.zeros((batch, g.num_kv_heads, g.page_size, g.head_dim),
                                  dtype=torch.float16, device=dev)})

    @classmethod
    def from_tensors(cls, geo: Q8Geometry, tensors: dict) -> "PagedQ8Cache":
        """Wrap existing pool and tail tensors (keys k_code ... v_tail)."""
        geo.check()
        c = cls.__new__(cls)
        c._set(geo, tensors)
        return c

    def _set(self, geo: Q8Geometry, t: dict) -> None:
        g = geo
        batch = t["k_tail"].shape[0]
        _check(batch >= 1, "batch must be positive")
        codes = (g.num_pages, g.num_kv_heads)
        want = {"k_code": ((*codes, g.page_size, g.head_dim), torch.uint8),
                "v_code": ((*codes, g.head_dim, g.page_size), torch.uint8),
                "k_scale": (codes, torch.float32), "v_scale": (codes, torch.float32),
                "k_tail": ((batch, g.num_kv_heads, g.page_size, g.head_dim), torch.float16),
                "v_tail": ((batch, g.num_kv_heads, g.page_size, g.head_dim), torch.float16)}
        for n, (shape, dtype) in want.items():
            check_shape(t[n], shape, n)
            _check(t[n].dtype == dtype and t[n].is_contiguous(), n, " must be contiguous ", dtype)
            _check(t[n].device == t["k_code"].device, n, " must be on the device of k_code")
        vars(self).update({n: t[n] for n in POOL}, geo=geo)
        self.batch, self.device = batch, t["k_code"].device
        self._index = self.device.index if self.device.type == "cuda" else -1
        self._record = _Pool(*(t[n].data_ptr() for n in POOL))
        self._pool = ctypes.byref(self._record)
        # what a call's tensors are compared with, and the workspace sizes asked for so far
        self._q_row, self._kv_row = (g.num_heads, g.head_dim), (g.num_kv_heads, g.head_dim)
        self._lens_shape, self._table_shape = (batch,), (batch, g.max_pages_per_seq)
        self._sizes = {}

    def __setattr__(self, name: str, value) -> None:
        """Another tensor in a tensor's place, or another geometry: checked, and what the calls
        hold goes by it."""
        if (name in POOL or name == "geo") and name in vars(self):
            t = {n: getattr(self, n) for n in POOL}
            if name == "geo":
                value.check()
                self._set(value, t)
            else:
                self._set(self.geo, {**t, name: value})
        else:
            object.__setattr__(self, name, value)

    def __getstate__(self):  # copies and pickles carry the tensors, not their addresses
        return {n: getattr(self, n) for n in ("geo", *POOL)}

    def __setstate__(self, state: dict) -> None:
        state["geo"].check()
        self._set(state["geo"], state)

    def sequence_view(self, b: int) -> "PagedQ8Cache":
        """A one-sequence cache sharing this cache's pool and sequence b's tail."""
        _check(0 <= b < self.batch, "a sequence must be in [0, ", self.batch, "), got ", b)
        t = {n: getattr(self, n) for n in POOL}
        t["k_tail"], t["v_tail"] = self.k_tail[b:b + 1], self.v_tail[b:b + 1]
        return PagedQ8Cache.from_tensors(self.geo, t)

    def pool(self):
        return tuple(getattr(self, n) for n in POOL)

    # ---- checks ----

    def _here(self, *named) -> None:
        for name, t in named:
            if t is not None:
                _check(t.device == self.device, name, " must be on the cache's device ",
                       self.device, ", got ", t.device)
        _check(self.device.type == "cuda", "the cache must be on a GPU device, got ", self.device)

    def _ints(self, t: torch.Tensor, n: int, name: str) -> None:
        check_shape(t, (n,), name)
        _check(t.dtype == torch.int32 and t.is_contiguous(), name, " must be contiguous int32")

    def _tables(self, lens, tables, name="SEQ_LENS") -> None:
        self._ints(lens, self.batch, name)
        check_shape(tables, (self.batch, self.geo.max_pages_per_seq), "BLOCK_TABLES")
        _check(tables.dtype == torch.int32 and tables.is_contiguous(),
               "BLOCK_TABLES must be contiguous int32")

    def _rows(self, t: torch.Tensor, heads: int, name: str) -> None:
        hd = self.geo.head_dim
        _check(t.dim() == 3 and t.shape[1:] == (heads, hd), name, " must be [tokens, ", heads,
               ", ", hd, "], got ", tuple(t.shape))
        _check(t.dtype in (torch.float16, torch.bfloat16), name, " must be fp16 or bf16")
        _check(t.shape[0] == 0 or (t.stride(2) == 1 and t.stride(1) == hd), name,
               " must have its heads side by side")
        _check(t.shape[0] <= 1 or t.stride(0) >= heads * hd, name,
               " must have a token's row after the one before")

    def _stride(self, t: torch.Tensor, heads: int) -> int:
        return t.stride(0) if t.shape[0] > 1 else heads * self.geo.head_dim

    def _weights(self, w: torch.Tensor, name="WEIGHTS") -> None:
        check_shape(w, (self.batch, self.geo.max_pages_per_seq), name)
        _check(w.dtype == torch.float32 and w.is_contiguous(), name, " must be contiguous fp32")

    # The checks of a call in one expression each: the named ones take the host longer than a
    # small call takes the GPU.  A call that fails one goes to the named checks, which say why.

    def _fits(self, lens: torch.Tensor, tables: torch.Tensor) -> bool:
        return (lens.shape == self._lens_shape and lens.dtype is torch.int32
                and lens.is_contiguous() and tables.shape == self._table_shape
                and tables.dtype is torch.int32 and tables.is_contiguous()
                and lens.get_device() == self._index == tables.get_device())

    def _fits_rows(self, t: torch.Tensor, row: tuple) -> bool:
        shape, dtype = t.shape, t.dtype
        return (len(shape) == 3 and shape[1] == row[0] and shape[2] == row[1]
                and t.is_contiguous() and (dtype is torch.float16 or dtype is torch.bfloat16)
                and t.get_device() == self._index)

    def _call(self, fn, *args) -> None:
        """The call with the cache's device current, on its current stream."""
        if torch._C._cuda_getDevice() == self._index:
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(self._index))
        else:
            with torch.cuda.device(self._index):
                rc = fn(*args, torch._C._cuda_getCurrentRawStream(self._index))
        if rc != 0:
            raise KiviLaunchError(last_error())

    def _workspace_size(self, key: tuple) -> int:
        if len(self._sizes) > 4096:
            self._sizes.clear()
        with torch.cuda.device(self._index):  # the size goes by its compute units
            size = self._sizes[key] = _lib.jacq_q8_attend_workspace_size(
                self.geo.ref, self.batch, *key)
        return size

    # ---- calls ----

    def append(self, new_k: torch.Tensor, new_v: torch.Tensor, block_tables: torch.Tensor,
               start_lens: torch.Tensor, cu_new: torch.Tensor | None = None,
               max_new: int | None = None) -> None:
        """Append new_k, new_v [tokens, NKV, HD] at start_lens [batch]: one token per
        sequence, or rows cu_new[b] to cu_new[b + 1] of sequence b (cu_new [batch + 1]
        int32), none with more than max_new (by default as many as there are rows).  Blocks
        that become full are quantised to the pages that block_tables names; tokens past
        the table's capacity are dropped.  The first block of a sequence's new tokens takes
        its tail in, so appending the same tokens twice is not the same as once."""
        nkv = self.geo.num_kv_heads
        total = new_k.shape[0] if new_k.dim() else 0
        fits = (self._index >= 0 and self._fits_rows(new_k, self._kv_row)
                and new_v.shape == new_k.shape and new_v.is_contiguous()
                and new_v.dtype is new_k.dtype and new_v.get_device() == self._index
                and self._fits(start_lens, block_tables))
        contiguous = fits
        if not fits:
            self._rows(new_k, nkv, "NEW_K")
            self._rows(new_v, nkv, "NEW_V")
            _check(new_v.shape[0] == total and new_v.dtype == new_k.dtype,
                   "NEW_V must have NEW_K's tokens and type")
            self._tables(start_lens, block_tables, "START_LENS")
        if cu_new is None:
            _check(total == self.batch, "without CU_NEW there is one new token per sequence: ",
                   self.batch, ", got ", total)
            _check(max_new is None or max_new == 1, "MAX_NEW is for CU_NEW")
            max_new = 1
        else:
            self._ints(cu_new, self.batch + 1, "CU_NEW")
            _check(max_new is None or max_new >= 0, "MAX_NEW must not be negative")
            max_new = total if max_new is None else min(int(max_new), total)
            fits = fits and cu_new.get_device() == self._index
        if not fits:
            self._here(("NEW_K", new_k), ("NEW_V", new_v), ("START_LENS", start_lens),
                       ("BLOCK_TABLES", block_tables), ("CU_NEW", cu_new))
        if contiguous:
            k_stride = v_stride = nkv * self.geo.head_dim
        else:
            k_stride, v_stride = self._stride(new_k, nkv), self._stride(new_v, nkv)
        self._call(_lib.jacq_q8_append, self.geo.ref, self._pool, new_k.data_ptr(),
                   new_v.data_ptr(), DTYPES[new_k.dtype], k_stride, v_stride, _ptr(cu_new),
                   start_lens.data_ptr(), block_tables.data_ptr(), total, max_new, self.batch)

    def _attend(self, q, cu_q, max_q, seq_lens, block_tables, window, sinks, scale, weights, decay,
                out, lse, workspace) -> torch.Tensor:
        g = self.geo
        nh, hd = self._q_row
        fits = (self._index >= 0 and self._fits_rows(q, self._q_row)
                and self._fits(seq_lens, block_tables))
        if not fits:
            self._rows(q, nh, "Q")
            self._tables(seq_lens, block_tables)
        total = q.shape[0]
        contiguous = fits
        if weights is not None:
            self._weights(weights)
            _check(max_q <= MAX_WEIGHTED_QUERIES, "WEIGHTS take at most ", MAX_WEIGHTED_QUERIES,
                   " queries per sequence, got ", max_q)
            _check(0.0 <= decay < math.inf, "DECAY must be finite and not negative")
        max_q = min(max_q, total)
        if window is None:
            window = 0
        else:
            _check(window >= 1, "WINDOW must be positive, or None")
        _check(sinks >= 0, "SINKS must not be negative")
        scale = hd ** -0.5 if scale is None else float(scale)
        _check(0.0 < scale < math.inf, "SCALE must be positive and finite")
        if cu_q is not None:
            self._ints(cu_q, self.batch + 1, "CU_Q")
        if out is None:  # empty_like is the quicker one, for a q that is contiguous
            out = (torch.empty_like(q) if contiguous else
                   torch.empty((total, nh, hd), dtype=q.dtype, device=q.device))
        else:
            check_shape(out, (total, nh, hd), "O")
            _check(out.dtype in (q.dtype, torch.float32) and out.is_contiguous(),
                   "O must be contiguous, of Q's type or fp32")
            fits = fits and out.get_device() == self._index
        if lse is not None:
            check_shape(lse, (total, nh), "LSE")
            _check(lse.dtype == torch.float32 and lse.is_contiguous(), "LSE must be contiguous fp32")
        if not (fits and cu_q is None and lse is None and weights is None and workspace is None):
            self._here(("Q", q), ("SEQ_LENS", seq_lens), ("BLOCK_TABLES", block_tables),
                       ("CU_Q", cu_q), ("O", out), ("LSE", lse), ("WEIGHTS", weights),
                       ("workspace", workspace))
        if workspace is None:
            key = (total, max_q, weights is not None)
            size = self._sizes.get(key)
            if size is None:
                size = self._workspace_size(key)
            if size:
                workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
        else:
            _check(workspace.is_contiguous(), "workspace must be contiguous")
            size = workspace.numel() * workspace.element_size()
        args = _ATTEND.pack(q.data_ptr(), _ptr(cu_q), seq_lens.data_ptr(), block_tables.data_ptr(),
                            out.data_ptr(), _ptr(lse), _ptr(weights),
                            nh * hd if contiguous else self._stride(q, nh),
                            DTYPES[q.dtype], DTYPES[out.dtype], self.batch, total, max_q,
                            min(window, 1 << 30), min(sinks, 1 << 30), scale, decay)
        self._call(_lib.jacq_q8_attend, g.ref, self._pool, args, _ptr(workspace), size)
        return out

    def decode(self, q: torch.Tensor, seq_lens: torch.Tensor, block_tables: torch.Tensor,
               window: int | None = None, sinks: int = 0, scale: float | None = None,
               weights: torch.Tensor | None = None, decay: float = 1.0,
               out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
        """q [batch, NH, HD], the last token of each sequence of seq_lens tokens -> O of q's
        type (or of ``out``'s, q's or fp32).

        window: a query sees the last ``window`` tokens, itself among them, and the first
        ``sinks`` of the sequence; None: all.  weights [batch, max_pages_per_seq] fp32 becomes
        decay * weights + the softmax weight of each block's tokens, summed over the heads;
        decay 0 overwrites; the call's workspace then takes, whatever the lengths are, 4 bytes
        for every head and every 16 tokens of the table's width (``prefill``: and query, the
        rows of a kv head rounded up).  lse [batch, NH] fp32 takes the log of the sum of
        exponentials.  A sequence of no tokens gives 0 (lse -inf)."""
        _check(q.dim() == 3 and q.shape[0] == self.batch, "Q must have one token per sequence (",
               self.batch, "), got ", tuple(q.shape))
        return self._attend(q, None, 1, seq_lens, block_tables, window, sinks, scale, weights,
                            decay, out, lse, workspace)

    def prefill(self, q: torch.Tensor, cu_q: torch.Tensor, max_q: int, seq_lens: torch.Tensor,
                block_tables: torch.Tensor, window: int | None = None, sinks: int = 0,
                scale: float | None = None, weights: torch.Tensor | None = None,
                decay: float = 1.0, out: torch.Tensor | None = None,
                lse: torch.Tensor | None = None, workspace: torch.Tensor | None = None
                ) -> torch.Tensor:
        """q [tokens, NH, HD]: rows cu_q[b] to cu_q[b + 1] (cu_q [batch + 1] int32) are the last
        tokens of sequence b, whose seq_lens[b] tokens are all in the cache; each sees the
        tokens up to its own, or the window and sinks of ``decode``.  No sequence has more than
        max_q: of one that has, the rows after its first max_q are left as they are, and so
        are rows outside every sequence (undefined in a fresh output).  weights, as in
        ``decode``, take at most 64 queries per sequence: the last ones of a prompt, in a call
        of their own."""
        _check(cu_q is not None, "CU_Q must be given")
        _check(max_q >= 0, "MAX_Q must not be negative")
        return self._attend(q, cu_q, int(max_q), seq_lens, block_tables, window, sinks, scale,
                            weights, decay, out, lse, workspace)

    def read(self, starts: torch.Tensor, ends: torch.Tensor, block_tables: torch.Tensor,
             total: int, dtype: torch.dtype = torch.float16):
        """The values of tokens starts[b] to ends[b] of each sequence, ends[b] its length, one
        sequence after another: K, V [total, NKV, HD].  total is their number: tokens past it
        are dropped, rows that none fills undefined."""
        g = self.geo
        fits = (self._index >= 0 and self._fits(ends, block_tables)
                and starts.shape == self._lens_shape and starts.dtype is torch.int32
                and starts.is_contiguous() and starts.get_device() == self._index)
        if not fits:
            self._tables(ends, block_tables, "ENDS")
            self._ints(starts, self.batch, "STARTS")
        _check(dtype in DTYPES, "values are read as fp16, bf16 or fp32, not ", dtype)
        _check(total >= 0, "TOTAL must not be negative")
        if not fits:
            self._here(("STARTS", starts), ("ENDS", ends), ("BLOCK_TABLES", block_tables))
        k = torch.empty((total, g.num_kv_heads, g.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        self._call(_lib.jacq_q8_read, g.ref, self._pool, starts.data_ptr(), ends.data_ptr(),
                   block_tables.data_ptr(), self.batch, total, k.data_ptr(), v.data_ptr(),
                   DTYPES[dtype])
        return k, v

    def evict(self, weights: torch.Tensor, seq_lens: torch.Tensor, block_tables: torch.Tensor,
              keep: int, sink_pages: int = 0, recent_pages: int = 0, out=None):
        """Evict the lightest blocks of each sequence that has more than ``keep`` full ones:
        the first sink_pages and the last recent_pages stay, of the others the heaviest (of
        equal ones the earlier, NaN lightest).  -> (block_tables, seq_lens, weights, evicted),
        new tensors or ``out``, which may hold the arguments themselves.

        A table row's kept entries move to its front; the evicted ones follow, so the
        sequence's next blocks reuse their pages unless the program takes them; no page is
        moved or copied.  Lengths count the tokens that are left."""
        fits = (self._index >= 0 and self._fits(seq_lens, block_tables)
                and weights.shape == self._table_shape and weights.dtype is torch.float32
                and weights.is_contiguous() and weights.get_device() == self._index)
        if not fits:
            self._tables(seq_lens, block_tables)
            self._weights(weights)
        _check(sink_pages >= 0 and recent_pages >= 0 and sink_pages + recent_pages <= keep,
               "KEEP must be at least SINK_PAGES + RECENT_PAGES, neither negative")
        if keep >= self.geo.max_pages_per_seq:  # no sequence has more
            keep, sink_pages, recent_pages = self.geo.max_pages_per_seq, 0, 0
        if out is None:
            out = (torch.empty_like(block_tables), torch.empty_like(seq_lens),
                   torch.empty_like(weights), torch.empty_like(seq_lens))
            tables_out, lens_out, weights_out, evicted = out
        else:
            tables_out, lens_out, weights_out, evicted = out
            self._tables(lens_out, tables_out, "the lengths given for output")
            self._weights(weights_out, "the weights given for output")
            self._ints(evicted, self.batch, "EVICTED")
            fits = False
        if not fits:
            self._here(("WEIGHTS", weights), ("SEQ_LENS", seq_lens), ("BLOCK_TABLES", block_tables),
                       *(("an output", t) for t in out))
        self._call(_lib.jacq_q8_evict, self.geo.ref, weights.data_ptr(), seq_lens.data_ptr(),
                   block_tables.data_ptr(), self.batch, keep, sink_pages, recent_pages,
                   tables_out.data_ptr(), lens_out.data_ptr(), weights_out.data_ptr(),
                   evicted.data_ptr())
        return out
