"""The 8-bit paged cache from its definition, in 64 bits: what the tests of jacq_amd.q8
compare with.  Tokens are kept as they came; blocks are quantised from the definition."""
from __future__ import annotations

import torch

FLOOR = 2.0 ** -24
TOP = {"int8": 127.0, "e4m3": 448.0}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def as_half(x):
    """What the cache holds of new values: fp16, saturated; NaN stays."""
    return torch.nan_to_num(x.double(), nan=float("nan"), posinf=65504.0,
                            neginf=-65504.0).clamp(-65504.0, 65504.0).half()


def couple_nan(k, v):
    """A NaN in a token's K or V of a kv head: its key is NaN, its V 0.  [..., HD]"""
    bad = (k.isnan() | v.isnan()).any(-1, keepdim=True)
    return torch.where(bad, torch.full_like(k, float("nan")), k), torch.where(
        bad, torch.zeros_like(v), v)


def e4m3(y):
    """Nearest value of 4 exponent and 3 mantissa bits (least exponent -6), ties to even."""
    _, e = torch.frexp(y)
    # from a table: torch's power functions are not exact on every device
    powers = torch.tensor([2.0 ** i for i in range(-9, 7)], dtype=y.dtype, device=y.device)
    step = powers[e.clamp(-5, 10).long() + 5]
    return (y / step).round() * step


def quantise(x, codes):
    """Blocks [..., P, HD] (fp16) -> code values (before the scale) and scales, in 64 bits."""
    x = x.double()
    a = torch.nan_to_num(x, nan=0.0).abs().amax((-2, -1)).clamp_min(FLOOR)
    y = x * TOP[codes] / a[..., None, None]
    y = y.round() if codes == "int8" else e4m3(y)
    poisoned = x.isnan().any(-1).any(-1)
    scale = torch.where(poisoned, torch.full_like(a, float("nan")), a / TOP[codes])
    return torch.where(poisoned[..., None, None], torch.zeros_like(y), y), scale


def code_bytes(y, codes):
    if codes == "int8":
        return (y + 128).to(torch.uint8)
    return y.float().to(torch.float8_e4m3fn).view(torch.uint8)


def byte_values(b, codes):
    if codes == "int8":
        return b.double() - 128
    return b.contiguous().view(torch.float8_e4m3fn).double()


def held_values(cache, tables, b, n):
    """K, V [NKV, n, HD] in 64 bits of sequence b, from the cache's tensors."""
    g = cache.geo
    full = n // g.page_size
    at = tables[b, :full].long()
    k = byte_values(cache.k_code[at], g.codes) * cache.k_scale[at].double()[..., None, None]
    v = byte_values(cache.v_code[at], g.codes) * cache.v_scale[at].double()[..., None, None]
    k = k.transpose(0, 1).reshape(g.num_kv_heads, -1, g.head_dim)
    v = v.transpose(2, 3).transpose(0, 1).reshape(g.num_kv_heads, -1, g.head_dim)
    left = n - full * g.page_size
    return (torch.cat((k, cache.k_tail[b, :, :left].double()), 1),
            torch.cat((v, cache.v_tail[b, :, :left].double()), 1))


def visible(pos, n, window, sinks, device):
    j = torch.arange(n, device=device)[None]
    pos = torch.as_tensor(pos, device=device)[:, None]
    see = j <= pos
    if window is not None:
        see = see & ((j < sinks) | (j > pos - window))
    return see


def attend(q, k, v, n, window=None, sinks=0, scale=None):
    """q [m, NH, HD], the last m of n tokens; k, v [NKV, n, HD] in 64 bits -> o, lse, p
    [NKV, m, G, n], and what tolerances are made of: sum(p |v|), the largest |v|, and the
    largest sum(|q| |k|) scale of a row."""
    m, nh, hd = q.shape
    nkv = k.shape[0]
    g = nh // nkv
    scale = hd ** -0.5 if scale is None else scale
    see = visible(range(n - m, n), n, window, sinks, q.device)[None, :, None]
    qq = q.double().view(m, nkv, g, hd).transpose(0, 1)  # [NKV, m, G, HD]
    x = torch.einsum("hmgd,hnd->hmgn", qq, k) * scale
    size = torch.einsum("hmgd,hnd->hmgn", qq.abs(), k.abs()) * abs(scale)
    x = torch.where(see, x, -torch.inf)
    lse = torch.logsumexp(x, -1) if n else torch.full((nkv, m, g), -torch.inf, device=q.device)
    p = torch.where(see, (x - torch.where(lse.isinf(), 0.0, lse)[..., None]).exp(), 0.0)
    vz = torch.where(see.any(1)[0, 0][None, :, None], v, 0.0) if m and n else v
    o = torch.einsum("hmgn,hnd->hmgd", p, vz)
    a = torch.einsum("hmgn,hnd->hmgd", p, vz.abs())
    size = torch.where(see, size, 0.0).amax(-1) if n else torch.zeros_like(lse)
    vmax = vz.abs().amax() if n else torch.zeros((), dtype=torch.float64, device=q.device)

    def rows(t):
        return t.transpose(0, 1).reshape(m, nh, *t.shape[3:])

    return {"o": rows(o), "lse": rows(lse), "p": p, "abs": rows(a), "size": rows(size),
            "vmax": vmax, "n": n}


def score_error(r, hd):
    """Relative error of a softmax weight from its score: an fp32 sum of HD products and a few
    roundings of the exponent, both against the largest sum(|q| |k|), and the row's own
    normalisation (twice).  The exponent also holds log2 of a scale: |.| <= 34, 2^-24 each."""
    return 2 * ((hd + 8) * 2.0 ** -24 * r["size"] + 64 * 2.0 ** -24)


def tolerance(r, hd, dtype):
    """Of an output: its own rounding, the weights' rounding to fp16 (half a step, relative; below
    2^-14 of the largest 2^-25 absolute), and the scores' error."""
    half = HALF_STEP[torch.float16]
    return (HALF_STEP[dtype] * r["o"].abs() + (half + score_error(r, hd)[..., None]) * r["abs"]
            * (1 + HALF_STEP[dtype]) + r["n"] * 2.0 ** -25 * r["vmax"] + 2.0 ** -25)


def assert_within(got, want, tol, what=""):
    got, nan = got.double(), want.isnan()
    assert torch.equal(got.isnan(), nan), f"{what}: NaN in other places"
    err = torch.where(nan, 0.0, (got - want).abs())
    err = torch.where(got == want, 0.0, err)  # equal infinities
    bad = ~(err <= torch.where(nan, 0.0, tol))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond tolerance, worst "
                           f"{float((err / tol).nan_to_num(0).max()):.2f} of it")


def evict(weights, lens, tables, page, keep, sink, recent):
    """Block by block: the lightest of the middle leave, of equal ones the last."""
    weights, tables, lens = weights.clone(), tables.clone(), list(lens)
    gone = []
    for b, n in enumerate(lens):
        full = n // page
        drop = max(0, full - keep)
        gone.append(drop)
        if not drop:
            continue
        w, t = weights[b].tolist(), tables[b].tolist()
        key = [float("-inf") if x != x else x for x in w]
        nan = [x != x for x in w]
        middle = sorted(range(sink, full - recent), key=lambda i: (not nan[i], key[i], -i))
        leave = sorted(middle[:drop])
        out = set(leave)
        stay = [i for i in range(full) if i not in out]
        tables[b, :full] = torch.tensor([t[i] for i in stay + leave])
        out = [w[i] for i in stay] + [0.0] * (len(w) - len(stay))
        if full < len(w):
            out[len(stay)] = w[full]
        weights[b] = torch.tensor(out)
        lens[b] = n - drop * page
    return tables, torch.tensor(lens, dtype=torch.int32), weights, torch.tensor(
        gone, dtype=torch.int32)
