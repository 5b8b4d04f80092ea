"""What the operators beside the int4 cache's writer and decode are measured on.

A program that serves a model from the int4 cache (32-token groups, K per channel, V per
token and 32 channels, the newest tokens in fp16) rotates the queries and keys of the new
tokens to their positions, appends them, and attends over the cache: with a chunk of a
prompt, with draft tokens, with one token under a sliding window; a decoder that hears an
encoder attends to all of its states, which a cache holds too.  To move or to check a
cache it reads its values back.

``own`` false computes all of it in plain torch; ``own`` true calls
``jacq_amd.kivi.PagedKiviCache`` and ``jacq_amd.rotary.Rotary``.

  prefill  ``new`` queries per sequence (all of a shorter one), its last tokens, each sees
           the tokens up to its own, or a window of them and the first ``sinks``
  cross    ``new`` queries per sequence over all of its tokens
  read     the values of each sequence's last ``span`` tokens (all of a shorter one)
  rotary   queries and keys of ``tokens`` rows of a fused projection

Lengths spread evenly over [lo, hi]; K has a few outlier channels per kv head, as the
workloads of jacq_amd.workloads have them.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
GROUP = 32
MOST_TOKENS = 6_000_000  # tokens x kv heads that a drawn case's cache holds
MOST_PAIRS = 1_300_000_000  # query x key pairs x query heads of a drawn case
MOST_ROTATED = 400_000_000  # values of a drawn rotary case


def case(op, nh, nkv, hd, batch, lo, hi, name=None, page=16, residual=128, dtype="fp16", **more):
    c = {"op": op, "nh": nh, "nkv": nkv, "hd": hd, "page": page, "residual": residual,
         "dtype": dtype, "batch": batch, "lo": lo, "hi": hi, **more}
    if name:
        c["name"] = name
    return c


def turn(nh, nkv, hd, tokens, lo, hi, name=None, dtype="fp16", part=1.0, layout="half",
         base=10000.0, scaling="none", factor=1.0, length=4096):
    c = {"op": "rotary", "nh": nh, "nkv": nkv, "hd": hd, "tokens": tokens, "lo": lo, "hi": hi,
         "dtype": dtype, "rd": 2 * max(1, int(hd * part) // 2), "layout": layout, "base": base,
         "scaling": scaling, "factor": factor, "length": length}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # two draft tokens of one user of a 1B model: latency alone
        case("prefill", 32, 4, 64, 1, 512, 512, "verify_one", residual=32, new=2),
        # a server's draft tokens: four queries of each sequence
        case("prefill", 40, 8, 128, 32, 1500, 6007, "verify_batch", new=4),
        # a server's decode step under a window and sinks: most of the cache is not looked at
        case("prefill", 32, 8, 128, 64, 1024, 16384, "window_decode", new=1, window=4096, sinks=4,
             dtype="bf16"),
        # a prompt from its first token
        case("prefill", 40, 8, 128, 1, 8191, 8191, "prompt", new=8191),
        # chunked prefill: four sequences at different places, odd chunk
        case("prefill", 32, 8, 128, 4, 4001, 16001, "chunk", new=511, page=32, dtype="bf16"),
        # ragged prompts under a window and sinks
        case("prefill", 14, 2, 64, 6, 700, 9001, "window_prompt", new=9001, window=1024, sinks=16),
        # a decoder's step over its encoders' states, each query head with keys of its own
        case("cross", 16, 16, 64, 32, 300, 1500, "cross_step", new=1, page=32, residual=32),
        # a decoder's prompt over long documents' states
        case("cross", 32, 8, 128, 8, 1001, 6000, "cross_prompt", new=333, dtype="bf16"),
        # a batch's caches moved to fp16
        case("read", 40, 8, 128, 16, 1024, 16384, "read_batch", span=16384),
        # what the writer left of the last tokens
        case("read", 14, 2, 64, 16, 2048, 2048, "read_recent", span=200, dtype="bf16"),
        # the rotation of a decode step of many users
        turn(40, 8, 128, 64, 1024, 16384, "rotary_step"),
        # a prompt's: part of the head, neighbouring pairs, frequencies slowed for long contexts
        turn(32, 8, 128, 8191, 0, 131071, "rotary_prompt", dtype="bf16", part=0.5,
             layout="interleaved", base=500000.0, scaling="turns", factor=8.0, length=8192),
    ]


# (query heads, kv heads, head dim) of the workloads and the tests
HEADS = ((32, 4, 64), (14, 2, 64), (24, 2, 64), (16, 16, 64), (32, 8, 128), (40, 8, 128),
         (20, 4, 128), (64, 8, 128), (32, 2, 128), (8, 8, 128))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("prefill", "prefill", "prefill", "cross", "cross", "read", "rotary"))
    nh, nkv, hd = rng.choice(HEADS)
    if op == "rotary":
        tokens = _log(rng, 1, 16384)
        while tokens * (nh + nkv) * hd > MOST_ROTATED:
            tokens = tokens * 3 // 4
        scaling = rng.choice(("none", "none", "linear", "base", "turns"))
        return turn(nh, nkv, hd, tokens, 0, _log(rng, 16, 1 << 20),
                    dtype=rng.choice(("fp16", "bf16", "fp32")), part=rng.choice((1.0, 0.5, 0.25)),
                    layout=rng.choice(("half", "interleaved")),
                    base=rng.choice((10000.0, 500000.0, 1000000.0)), scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0)),
                    length=rng.choice((4096, 8192)))
    more = {"page": rng.choice((16, 16, 32)), "residual": rng.choice((32, 64, 128, 128, 256)),
            "dtype": rng.choice(("fp16", "bf16"))}
    if op == "read":
        hi, batch = _log(rng, 16, 32768), _log(rng, 1, 64)
        while batch * hi * nkv > MOST_TOKENS // 4:
            batch, hi = max(1, batch * 3 // 4), max(16, hi * 3 // 4)
        return case(op, nh, nkv, hd, batch, max(1, hi // rng.choice((1, 4, 16))), hi,
                    span=rng.choice((hi, _log(rng, 1, hi))), **more)
    if op == "prefill" and rng.random() < 0.4:
        more["window"], more["sinks"] = _log(rng, 16, 8192), rng.choice((0, 1, 4, 16, 100))
    if op == "cross":
        new, hi, batch = _log(rng, 1, 2048), _log(rng, 8, 8192), _log(rng, 1, 64)
    else:
        kind = rng.choice(("one", "few", "many", "many"))
        new = {"one": 1, "few": rng.randint(2, 40), "many": _log(rng, 40, 8192)}[kind]
        batch = _log(rng, 1, 8 if kind == "many" else 128)
        hi = rng.choice((new, new + _log(rng, 16, 16384))) if kind == "many" else _log(rng, 24, 40000)
    while batch * hi * nkv > MOST_TOKENS or batch * new * hi * nh > MOST_PAIRS:
        if batch > 1:
            batch -= max(1, batch // 4)
        else:
            new, hi = max(1, new * 3 // 4), max(8, hi * 3 // 4)
    lo = rng.choice((hi, max(1, hi // 2), max(1, hi // 16)))
    return case(op, nh, nkv, hd, batch, lo, hi, new=min(new, hi) if op == "prefill" else new, **more)


# ---- sizes ----

def lengths(c):
    """One length per sequence, spread over [lo, hi] by the golden ratio."""
    lo, hi = c["lo"], c["hi"]
    return [lo + int((hi - lo + 1) * ((i + 1) * 0.6180339887498949 % 1)) for i in range(c["batch"])]


def queries(c, n):
    """Queries of a sequence of n tokens."""
    return min(n, c["new"]) if c["op"] == "prefill" else c["new"]


def old_tokens(c, n):
    """How many of n tokens are int4: whole groups, with at least `residual` left in fp16."""
    return max(0, n - c["residual"]) // GROUP * GROUP


def held_bytes(c, first, n):
    """Bytes that a kv head's tokens [first, n) take in the cache, K and V."""
    hd, old = c["hd"], old_tokens(c, n)
    quant = max(0, old - first)
    groups = -(-quant // GROUP)
    return (quant * (hd + 4 * hd // 32) + groups * 4 * hd + (n - max(first, old)) * 4 * hd)


def work(c):
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "rotary":
        values = c["tokens"] * (nh + nkv) * hd
        return {"bytes": values * 2 * size + 4 * c["tokens"],
                "flops": c["tokens"] * (nh + nkv) * c["rd"] * 3}
    total = flops = 0
    for n in lengths(c):
        if c["op"] == "read":
            first = n - min(n, c["span"])
            total += nkv * held_bytes(c, first, n) + 4 * (old_tokens(c, n) // c["page"])
            total += 2 * (n - first) * nkv * hd * size
            flops += 4 * (n - first) * nkv * hd
            continue
        m, window, sinks = queries(c, n), c.get("window"), c.get("sinks", 0)
        lo = max(0, n - m + 1 - window) if window else 0
        total += nkv * (held_bytes(c, lo, n) + min(sinks, lo) * (hd + 4 * hd // 32))
        total += 4 * ((n - lo) // c["page"]) + m * nh * hd * 2 * size
        if c["op"] == "cross":
            flops += 4 * nh * hd * m * n
            continue
        for p in range(n - m, n):
            first = max(0, p + 1 - window) if window else 0
            flops += 4 * nh * hd * (p + 1 - first + min(sinks, first))
    return {"bytes": total, "flops": flops}


def speeds(c):
    """Radians a position of each pair, and the factor on cosine and sine."""
    rd, base, factor = c["rd"], c["base"], c["factor"]
    if c["scaling"] == "base":  # the slowest pair by the factor, the fastest not at all
        base *= factor ** (rd / max(1, rd - 2))
    f = [base ** (-2 * i / rd) for i in range(rd // 2)]
    if c["scaling"] == "linear":
        return [x / factor for x in f], 1.0
    if c["scaling"] == "turns":
        # pairs with fewer than 1 turn over the length by the factor, with more than 32 not
        out = []
        for x in f:
            s = min(1.0, max(0.0, (c["length"] * x / (2 * math.pi) - 1.0) / 31.0))
            out.append(x * (s + (1.0 - s) / factor))
        return out, 0.1 * math.log(factor) + 1.0
    return f, 1.0


# ---- the plain form ----

def unpack(b):
    """Two codes a byte, the low half first."""
    return torch.stack((b & 15, b >> 4), -1).flatten(-2).float()


def rows(c, s, b, n):
    """K and V [kv heads, n, HD] of sequence b, as the cache holds them."""
    page, hd, nkv = c["page"], c["hd"], c["nkv"]
    old = old_tokens(c, n)
    at = s["tables"][b, :old // page].long()
    first = s["tables"][b, :old // page:GROUP // page].long()  # a group's first page
    k = unpack(s["k_code"][at]).transpose(0, 1).reshape(nkv, -1, GROUP, hd)
    k = (k * s["k_scale"][first].float().transpose(0, 1)[:, :, None]
         + s["k_zero"][first].float().transpose(0, 1)[:, :, None]).reshape(nkv, old, hd)
    v = unpack(s["v_code"][at]).transpose(0, 1).reshape(nkv, old, hd // 32, 32)
    v = (v * s["v_scale"][at].float().transpose(0, 1).reshape(nkv, old, hd // 32, 1)
         + s["v_zero"][at].float().transpose(0, 1).reshape(nkv, old, hd // 32, 1))
    return (torch.cat((k, s["k_scr"][b, :, :n - old].float()), 1),
            torch.cat((v.reshape(nkv, old, hd), s["v_scr"][b, :, :n - old].float()), 1))


def plain_attend(c, s):
    g, hd = c["nh"] // c["nkv"], c["hd"]
    out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=s["q"].device)
    at = 0
    for b, n in enumerate(s["lens"]):
        m = queries(c, n)
        k, v = rows(c, s, b, n)
        hidden = None
        if c["op"] == "prefill":
            pos = torch.arange(n - m, n, device=k.device)[:, None]
            j = torch.arange(n, device=k.device)[None]
            hidden = j > pos
            if c.get("window"):
                hidden |= (j <= pos - c["window"]) & (j >= c["sinks"])
            hidden = hidden[:, None]
        for h in range(c["nkv"]):
            q = s["q"][at:at + m, h * g:(h + 1) * g].float()
            x = torch.matmul(q, k[h].t().contiguous()) / math.sqrt(hd)
            if hidden is not None:
                x = x.masked_fill(hidden, float("-inf"))
            p = (x - x.amax(2, keepdim=True)).exp()
            p = p / p.sum(2, keepdim=True)
            out[at:at + m, h * g:(h + 1) * g] = torch.matmul(p, v[h]).to(out.dtype)
        at += m
    return out


def plain_read(c, s):
    ks, vs = [], []
    for b, n in enumerate(s["lens"]):
        k, v = rows(c, s, b, n)
        first = n - min(n, c["span"])
        ks.append(k[:, first:].transpose(0, 1).to(DTYPE[c["dtype"]]))
        vs.append(v[:, first:].transpose(0, 1).to(DTYPE[c["dtype"]]))
    return torch.cat(ks), torch.cat(vs)


def plain_rotary(c, s):
    # 64 bits for the angle: far positions lose its digits in 32
    angle = s["positions"].double()[:, None] * s["speeds"]
    cos, sin = angle.cos().float() * s["amplitude"], angle.sin().float() * s["amplitude"]
    cos, sin, rd = cos[:, None], sin[:, None], c["rd"]
    res = []
    for x in (s["q"], s["k"]):
        y = x.float().clone()
        if c["layout"] == "half":
            a, b = y[..., :rd // 2].clone(), y[..., rd // 2:rd].clone()
            y[..., :rd // 2], y[..., rd // 2:rd] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = y[..., 0:rd:2].clone(), y[..., 1:rd:2].clone()
            y[..., 0:rd:2], y[..., 1:rd:2] = a * cos - b * sin, b * cos + a * sin
        res.append(y.to(x.dtype))
    return tuple(res)


# ---- what a program has in hand ----

def quantise(x, dim):
    """x in 16 levels between its least and largest value along dim -> codes, scale, zero."""
    lo = x.amin(dim, keepdim=True)
    scale = (x.amax(dim, keepdim=True) - lo) / 15
    code = ((x - lo) / scale.clamp_min(1e-30)).round().clamp(0, 15).to(torch.uint8)
    return code, scale.half().squeeze(dim), lo.half().squeeze(dim)


def pack(code):
    return code[..., 0::2] | code[..., 1::2] << 4


def prepare_rotary(c, gen):
    nh, nkv, hd, tokens = c["nh"], c["nkv"], c["hd"], c["tokens"]
    # one projection's output: a token's queries, keys and values side by side
    qkv = torch.randn((tokens, (nh + 2 * nkv) * hd), generator=gen, device="cuda").to(
        DTYPE[c["dtype"]])
    s = {"case": c, "qkv": qkv}
    s["q"] = qkv[:, :nh * hd].unflatten(1, (nh, hd))
    s["k"] = qkv[:, nh * hd:(nh + nkv) * hd].unflatten(1, (nkv, hd))
    first = int(torch.randint(c["lo"], max(c["lo"], c["hi"] - tokens) + 1, (1,), generator=gen,
                              device="cuda"))
    if tokens > 256:  # a prompt's positions
        s["positions"] = torch.arange(first, first + tokens, dtype=torch.int32, device="cuda")
    else:  # a token each of as many sequences
        s["positions"] = torch.randint(c["lo"], c["hi"] + 1, (tokens,), generator=gen,
                                       device="cuda", dtype=torch.int32)
    f, s["amplitude"] = speeds(c)
    s["speeds"] = torch.tensor(f, dtype=torch.float64, device="cuda")
    if own:
        from jacq_amd import rotary
        s["rotary"] = rotary.Rotary(
            hd, rotary_dim=c["rd"], base=c["base"], layout=c["layout"],
            scaling=None if c["scaling"] == "none" else rotary.Scaling(
                c["scaling"], c["factor"], length=c["length"], slow=1.0, fast=32.0))
    return s


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] == "rotary":
        return prepare_rotary(c, gen)
    nkv, hd, page, batch, op = c["nkv"], c["hd"], c["page"], c["batch"], c["op"]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    outliers = torch.rand((nkv, hd), generator=gen, device="cuda").argsort(1)[:, :hd // 16]
    k_chan = torch.ones((nkv, hd), device="cuda").scatter_(1, outliers, 6.0)
    order = torch.randperm(batch, generator=gen, device="cuda").tolist()
    even = lengths(c)
    lens = [even[i] for i in order]
    per = GROUP // page  # pages of a group
    need = [-(-n // GROUP) * per for n in lens]
    width, pages = max(need), sum(need)
    perm = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    tables = torch.zeros((batch, width), dtype=torch.int32, device="cuda")
    at = 0
    for b, k in enumerate(need):
        tables[b, :k] = perm[at:at + k]
        at += k
    s = {"case": c, "lens": lens, "tables": tables,
         "seq_lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    half = torch.float16
    for x in ("k", "v"):
        s[x + "_code"] = torch.empty((pages, nkv, page, hd // 2), dtype=torch.uint8, device="cuda")
    s["k_scale"] = torch.empty((pages, nkv, hd), dtype=half, device="cuda")
    s["v_scale"] = torch.empty((pages, nkv, page, hd // 32), dtype=half, device="cuda")
    s["k_zero"], s["v_zero"] = torch.empty_like(s["k_scale"]), torch.empty_like(s["v_scale"])
    step = max(1, (1 << 25) // (nkv * GROUP * hd))
    groups = perm.long().view(-1, per)  # the pages of each group
    for g0 in range(0, groups.shape[0], step):
        at = groups[g0:g0 + step]
        n = at.shape[0]
        code, scale, zero = quantise(randn(n, nkv, GROUP, hd) * k_chan[:, None], 2)
        code = pack(code).view(n, nkv, per, page, hd // 2)
        vcode, vscale, vzero = quantise(randn(n, nkv, GROUP, hd // 32, 32), 4)
        vcode = pack(vcode.flatten(3)).view(n, nkv, per, page, hd // 2)
        vscale, vzero = (t.view(n, nkv, per, page, hd // 32) for t in (vscale, vzero))
        for i in range(per):
            p = at[:, i]
            s["k_code"][p], s["k_scale"][p], s["k_zero"][p] = code[:, :, i], scale, zero
            s["v_code"][p], s["v_scale"][p], s["v_zero"][p] = (
                vcode[:, :, i], vscale[:, :, i], vzero[:, :, i])
    rs = c["residual"] + GROUP
    s["k_scr"] = (randn(batch, nkv, rs, hd) * k_chan[:, None]).half()
    s["v_scr"] = randn(batch, nkv, rs, hd).half()
    if op == "read":
        firsts = [n - min(n, c["span"]) for n in lens]
        s["firsts"] = torch.tensor(firsts, dtype=torch.int32, device="cuda")
        s["total"] = sum(lens) - sum(firsts)
    else:
        m = [queries(c, n) for n in lens]
        s["q"] = randn(sum(m), c["nh"], hd).to(DTYPE[c["dtype"]])
        cu = [0]
        for x in m:
            cu.append(cu[-1] + x)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        s["max_q"] = max(m)
    if own:
        from jacq_amd import kivi
        geo = kivi.KiviGeometry(c["nh"], nkv, hd, page, GROUP, c["residual"], width, pages)
        s["cache"] = kivi.PagedKiviCache.from_tensors(geo, {
            n: s[n] for n in ("k_code", "k_scale", "k_zero", "v_code", "v_scale", "v_zero",
                              "k_scr", "v_scr")})
    return s


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"read": plain_read, "rotary": plain_rotary}.get(op, plain_attend)(c, s)
    if op == "rotary":
        return s["rotary"].rotate(s["q"], s["k"], s["positions"])
    cache = s["cache"]
    if op == "read":
        return cache.read(s["firsts"], s["seq_lens"], s["tables"], s["total"],
                          dtype=DTYPE[c["dtype"]])
    if op == "cross":
        return cache.cross(s["q"], s["cu"], s["max_q"], s["seq_lens"], s["tables"])
    seen = {"window": c["window"], "sinks": c["sinks"]} if c.get("window") else {}
    return cache.prefill(s["q"], s["cu"], s["max_q"], s["seq_lens"], s["tables"], **seen)


# ---- the definition in 64 bits ----

def value64(c, s, b, h, n):
    """K and V [n, HD] of a kv head of a sequence, token by token of the table, in 64 bits."""
    page, hd = c["page"], c["hd"]
    old = old_tokens(c, n)
    t = torch.arange(old, device="cuda")
    pages, inside = s["tables"][b].long()[t // page], t % page
    group = s["tables"][b].long()[t // GROUP * GROUP // page]
    d = torch.arange(hd, device="cuda")
    shift = 4 * (d % 2)
    res = []
    for x in ("k", "v"):
        code = (s[x + "_code"][pages, h, inside].long()[:, d // 2] >> shift) % 16
        if x == "k":
            scale, zero = s["k_scale"][group, h], s["k_zero"][group, h]
        else:
            scale = s["v_scale"][pages, h, inside][:, d // 32]
            zero = s["v_zero"][pages, h, inside][:, d // 32]
        old_part = code.double() * scale.double() + zero.double()
        res.append(torch.cat((old_part, s[x + "_scr"][b, h, :n - old].double())))
    return res


def exact_rotary(c, s):
    f = torch.tensor(speeds(c)[0], dtype=torch.float64, device="cuda")
    phase = torch.outer(s["positions"].double(), f)
    spin = torch.polar(torch.full_like(phase, speeds(c)[1]), phase)[:, None]
    rd, res = c["rd"], []
    for x in (s["q"], s["k"]):
        turned = x[..., :rd].double()
        if c["layout"] == "half":
            turned = turned.unflatten(-1, (2, rd // 2)).transpose(-1, -2)
        else:
            turned = turned.unflatten(-1, (rd // 2, 2))
        turned = torch.view_as_real(torch.view_as_complex(turned.contiguous()) * spin)
        if c["layout"] == "half":
            turned = turned.transpose(-1, -2)
        res.append(torch.cat((turned.flatten(-2), x[..., rd:].double()), -1))
    return tuple(res)


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rotary":
        return exact_rotary(c, s)
    nkv, hd = c["nkv"], c["hd"]
    g = c["nh"] // nkv
    outs, ks, vs, at = [], [], [], 0
    for b, n in enumerate(s["lens"]):
        if c["op"] == "read":
            both = [value64(c, s, b, h, n) for h in range(nkv)]
            first = n - min(n, c["span"])
            ks.append(torch.stack([k[first:] for k, _ in both], 1))
            vs.append(torch.stack([v[first:] for _, v in both], 1))
            continue
        m = queries(c, n)
        heads = []
        for h in range(nkv):
            k, v = value64(c, s, b, h, n)
            kt = k.t().contiguous()
            got = []
            for i0 in range(0, m, 512):  # queries a few at a time: a prompt's scores are large
                i1 = min(m, i0 + 512)
                q = s["q"][at + i0:at + i1, h * g:(h + 1) * g].double()
                x = torch.matmul(q.reshape(-1, hd), kt).view(i1 - i0, g, n) * hd ** -0.5
                if c["op"] == "prefill":
                    pos = torch.arange(n - m + i0, n - m + i1, device="cuda").view(-1, 1, 1)
                    j = torch.arange(n, device="cuda").view(1, 1, -1)
                    see = j <= pos
                    if c.get("window"):
                        see &= (j > pos - c["window"]) | (j < c["sinks"])
                    x = torch.where(see, x, -math.inf)
                p = torch.softmax(x, 2)
                got.append(torch.matmul(p.reshape(-1, n), v).view(i1 - i0, g, hd))
            heads.append(torch.cat(got))
        outs.append(torch.cat(heads, 1))
        at += m
    if c["op"] == "read":
        return torch.cat(ks), torch.cat(vs)
    return torch.cat(outs)
