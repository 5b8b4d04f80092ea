"""The int4 cache's attention of chunks and its read-back from their definition, in 64 bits."""
from __future__ import annotations

import numpy as np
import torch

from tests.q8_ref import HALF_STEP, assert_within  # noqa: F401

GROUP = 32


def old_tokens(geo, n):
    cap = geo.max_pages_per_seq * geo.page_size // GROUP * GROUP
    return min(max(0, n - geo.residual) // GROUP * GROUP, cap)


def to_half(x):
    """64 bits to fp16 in one rounding (torch's own goes through 32)."""
    with np.errstate(over="ignore"):
        return torch.from_numpy(x.cpu().numpy().astype(np.float16)).to(x.device)


def unpack(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2).double()


def exact_values(cache, tables, b, n):
    """K, V [NKV, n, HD] in 64 bits of sequence b, and whether each token's page is there (its
    group's first page, for K's scales, too)."""
    g = cache.geo
    old, nkv, hd, page = old_tokens(g, n), g.num_kv_heads, g.head_dim, g.page_size
    at = tables[b, :old // page].long()
    known = (at >= 0) & (at < g.num_pages)
    at = torch.where(known, at, 0)
    first = at[::GROUP // page]
    there = known.repeat_interleave(page) & known[::GROUP // page].repeat_interleave(GROUP)

    def heads(x):  # [pages, NKV, ...] -> [NKV, pages, ...]
        return x.transpose(0, 1)

    k = heads(unpack(cache.k_code[at])).reshape(nkv, -1, GROUP, hd)
    k = (k * heads(cache.k_scale[first].double())[:, :, None]
         + heads(cache.k_zero[first].double())[:, :, None]).reshape(nkv, old, hd)
    v = heads(unpack(cache.v_code[at])).reshape(nkv, old, hd // 32, 32)
    v = (v * heads(cache.v_scale[at].double()).reshape(nkv, old, hd // 32, 1)
         + heads(cache.v_zero[at].double()).reshape(nkv, old, hd // 32, 1)).reshape(nkv, old, hd)
    there = torch.cat((there, torch.ones(n - old, dtype=torch.bool, device=there.device)))
    return (torch.cat((k, cache.k_scr[b, :, :n - old].double()), 1),
            torch.cat((v, cache.v_scr[b, :, :n - old].double()), 1), there)


def held_values(cache, tables, b, n):
    """K, V as the products take them: rounded to fp16; a token whose V is not finite, or whose page
    is not there, has a NaN key and a V of 0."""
    k, v, there = exact_values(cache, tables, b, n)
    k, v = to_half(k).double(), to_half(v).double()
    bad = (~v.isfinite()).any(-1, keepdim=True) | ~there[None, :, None]
    return torch.where(bad, torch.nan, k), torch.where(bad, 0.0, v)


def visible(m, n, window, sinks, causal, device):
    j = torch.arange(n, device=device)[None]
    pos = torch.arange(n - m, n, device=device)[:, None]
    see = j <= pos if causal else torch.ones((m, n), dtype=torch.bool, device=device)
    if window is not None:
        see = see & ((j < sinks) | (j > pos - window))
    return see


def attend(q, k, v, window=None, sinks=0, causal=True, scale=None):
    """q [m, NH, HD]; k, v [NKV, n, HD] in 64 bits -> o, lse, and what tolerances are made of:
    sum(p |v|), the largest sum(|q| |k|) scale of a row, the largest |v|."""
    m, nh, hd = q.shape
    nkv, n = k.shape[:2]
    g = nh // nkv
    scale = hd ** -0.5 if scale is None else scale
    qq = q.double().view(m, nkv, g, hd).transpose(0, 1).reshape(nkv, m * g, hd)
    see = visible(m, n, window, sinks, causal, q.device).repeat_interleave(g, 0)[None]
    kt = k.transpose(1, 2).contiguous()
    x = torch.matmul(qq, kt) * scale
    size = torch.matmul(qq.abs(), kt.abs()) * scale
    x = torch.where(see, x, -torch.inf)
    size = torch.where(see, size, 0.0).amax(-1) if n else torch.zeros(nkv, m * g, device=q.device)
    lse = (torch.logsumexp(x, -1) if n else
           torch.full((nkv, m * g), -torch.inf, dtype=torch.float64, device=q.device))
    p = torch.where(see, (x - torch.where(lse.isinf(), 0.0, lse)[..., None]).exp(), 0.0)
    o, a = torch.matmul(p, v), torch.matmul(p, v.abs())
    vmax = v.abs().amax() if n else torch.zeros((), dtype=torch.float64, device=q.device)

    def rows(t):
        return t.reshape(nkv, m, g, *t.shape[2:]).transpose(0, 1).reshape(m, nh, *t.shape[2:])

    return {"o": rows(o), "lse": rows(lse), "abs": rows(a), "size": rows(size), "vmax": vmax, "n": n}


def score_error(r, hd):
    """Relative error of a softmax weight from its score: an fp32 sum of HD products and a few
    roundings of the exponent (of up to 2^8 after the log2(e)), both against the largest
    sum(|q| |k|), and the row's own normalisation (twice)."""
    return 2 * ((hd + 8) * 2.0 ** -24 * r["size"] + 64 * 2.0 ** -24)


def tolerance(r, hd, dtype):
    """Of an output against held_values: its own rounding, the weights' rounding to fp16 (half a
    step, relative; below 2^-14 of the largest 2^-25 absolute), and the scores' error."""
    half = HALF_STEP[torch.float16]
    return (HALF_STEP[dtype] * r["o"].abs() + (half + score_error(r, hd)[..., None]) * r["abs"]
            * (1 + HALF_STEP[dtype]) + r["n"] * 2.0 ** -25 * r["vmax"] + 2.0 ** -25)
