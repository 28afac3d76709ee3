"""Performance cases of the operators between a decoder's qkv and output projections, over a paged
key/value cache held in 4 bits, as a serving program runs them:

  rope    per-head RMSNorm of queries and keys with the rotation, one or several position axes
  append  the same with the new keys and values rounded into their cache slots, and the written
          tokens read back
  attn    attention over the cache: one token per sequence, a few drafted tokens, prompt chunks
  move    page copies over all layers and the remapped page table: forks and compaction

The cache's layout: [pages, kv heads, page / 16, 17 d] bytes, 16 tokens of one head at a time:
key codes [16][d/2], value codes [planes][4][16][4][bytes] (token 4 g + i; runs of 8 channels, 4 at
d = 64), key scales [16][d/32], value scales [d/32][16]. Codes are e2m1, the low nibble the even
channel; scales are biased exponents of a power of two for 32 channels of one token.

Head counts are those of the benchmark's 5120-hidden layer (qkv 10240 = 48 + 2 x 16 heads of 128),
of its 4096- and 3584-hidden neighbours (32 + 2 x 8, 28 + 2 x 4), and generic ones of 64 and 256.
"""
from __future__ import annotations

import functools
import math
import random

import torch

own = False

EPS = 1e-6
# name -> (query heads, kv heads, head size, rotated channels)
HEADS = {
    "h5120": (48, 16, 128, 128),
    "h4096": (32, 8, 128, 128),
    "h3584": (28, 4, 128, 128),
    "wide": (24, 4, 256, 64),           # wide heads, a quarter of each rotated
    "wide2": (16, 2, 256, 256),
    "small": (32, 32, 64, 64),          # every query head with keys of its own
    "small8": (64, 8, 64, 32),
}
TABLE = 32768                           # rows of the cos/sin table
CACHED_MAX = 48 * 4000 * 8 * 128        # cached tokens x kv heads x head size of the largest case
PRODUCTS_MAX = 4096 * 4096 * 32 * 128 // 2  # query-key pairs x heads x head size of the largest case


# ---- cases --------------------------------------------------------------------------------------
def listed():
    return [
        # one decoded token: the smallest call
        dict(name="rope_t1", op="rope", heads="h4096", T=1, axes=1, adjacent=False, gemma=True),
        # an image-and-text prompt of odd length: three axes, wide heads, a quarter rotated
        dict(name="rope_axes_t3777", op="rope", heads="wide", T=3777, axes=3, adjacent=False,
             gemma=True),
        # a decode batch of 61 sequences, one token each, at slots all over the cache
        dict(name="append_t61", op="append", heads="h4096", T=61, axes=1, adjacent=False,
             gemma=True, page=16, chunk=False),
        # a prefill chunk that begins in the middle of a page
        dict(name="append_t4096", op="append", heads="h5120", T=4096, axes=3, adjacent=False,
             gemma=False, page=64, chunk=True),
        # one sequence of a short context: the smallest attention
        dict(name="decode_b1_l500", op="attn", heads="h4096", B=1, Q=1, L=500, Lmin=500, page=16,
             window=0, mixed=False),
        # a decode batch of uneven contexts
        dict(name="decode_b48_l8000", op="attn", heads="h4096", B=48, Q=1, L=8000, Lmin=200,
             page=16, window=0, mixed=False),
        # one sequence of a very long context
        dict(name="decode_b1_l131072", op="attn", heads="h4096", B=1, Q=1, L=131072, Lmin=131072,
             page=64, window=0, mixed=False),
        # speculative verify: eight drafted tokens a sequence
        dict(name="verify_b8_q8_l4001", op="attn", heads="h5120", B=8, Q=8, L=4001, Lmin=1000,
             page=32, window=0, mixed=False),
        # a prompt of 4096 tokens in one chunk
        dict(name="prefill_4096", op="attn", heads="h4096", B=1, Q=4096, L=4096, Lmin=4096,
             page=64, window=0, mixed=False),
        # decode rows beside prompt chunks over long contexts, wide heads, a sliding window
        dict(name="chunks_wide_q513", op="attn", heads="wide", B=6, Q=513, L=9001, Lmin=600,
             page=32, window=4096, mixed=True),
        # a fork: the last, partly filled page of four sequences
        dict(name="move_n4", op="move", heads="h3584", layers=24, pages=300, page=32, n=4, B=8),
        # compaction of a fragmented pool
        dict(name="move_n600", op="move", heads="h4096", layers=24, pages=1600, page=16, n=600,
             B=32),
    ]


def _log(rng, lo, hi):
    n = max(lo, min(hi, int(round(2.0 ** rng.uniform(math.log2(lo), math.log2(hi))))))
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choices(["rope", "append", "attn", "move"], [3, 3, 8, 2])[0]
    heads = rng.choice(sorted(HEADS))
    Hq, Hkv, d, _ = HEADS[heads]
    page = rng.choice([16, 32, 64, 128])
    if op == "rope" or op == "append":
        most = min(4096, 4096 * 80 * 128 // ((Hq + 2 * Hkv) * d))
        case = dict(op=op, heads=heads, T=_log(rng, 1, most), axes=rng.choice([1, 1, 3, 2]),
                    adjacent=rng.random() < 0.25, gemma=rng.random() < 0.5)
        if op == "append":
            case.update(page=page, chunk=case["T"] > 16 and rng.random() < 0.6)
        return case
    if op == "move":
        pages = _log(rng, 40, 1600)
        layers = rng.randint(4, 24)
        most = (3 << 30) // (layers * page * Hkv * d * 17 // 16)
        pages = min(pages, max(40, most))
        most = (250 << 20) // (layers * page * Hkv * d * 17 // 16)
        n = max(1, min(_log(rng, 1, 600), pages // 3, most))
        return dict(op=op, heads=heads, layers=layers, pages=pages, page=page, n=n,
                    B=rng.randint(1, 32))
    kind = rng.choice(["decode", "decode", "verify", "prefill", "mixed"])
    B, Q, L, window = 1, 1, 1, 0
    if kind in ("decode", "verify"):
        Q = 1 if kind == "decode" else rng.randint(2, 9)
        B = _log(rng, 1, 64)
        L = _log(rng, 16, min(131072, max(64, CACHED_MAX // (B * Hkv * d))))
        Lmin = L if B == 1 else rng.randint(max(1, L // 40), L)
    elif kind == "prefill":
        Q = _log(rng, 17, 4096)
        B = max(1, min(_log(rng, 1, 8), 4096 // Q))
        most = PRODUCTS_MAX // (B * Q * Hq * d)
        L = Q + (rng.randint(0, min(8192, max(0, most - Q))) if rng.random() < 0.5 else 0)
        Lmin = rng.randint(max(1, Q // 2), L) if B > 1 else L
    else:
        Q, B = _log(rng, 33, 520), rng.randint(2, 8)
        most = max(600, PRODUCTS_MAX // (-(-B // 2) * Q * Hq * d))
        L = max(Q, _log(rng, 600, min(9001, most)))
        Lmin = min(L, 600)
    if rng.random() < 0.25:
        window = _log(rng, 64, 4096)
    return dict(op=op, heads=heads, B=B, Q=Q, L=L, Lmin=Lmin, page=page, window=window,
                mixed=kind == "mixed")


def _lens(case):
    """Cached tokens and query tokens of each sequence (the case's own, the same for every seed)."""
    r = random.Random("%d %d %d %d" % (case["B"], case["Q"], case["L"], case["Lmin"]))
    lens = [case["L"]] + [r.randint(case["Lmin"], case["L"]) for _ in range(case["B"] - 1)]
    qs = [1 if case["mixed"] and i % 2 else min(case["Q"], n) for i, n in enumerate(lens)]
    return lens, qs


def _pairs(n, q, window):
    """Query-key pairs of a sequence of n tokens whose last q ask."""
    if not window or window >= n:
        return q * n - q * (q - 1) // 2
    return sum(min(window, n - i) for i in range(q))


def work(case):
    Hq, Hkv, d, rot = HEADS[case["heads"]]
    if case["op"] in ("rope", "append"):
        T, elements = case["T"], case["T"] * (Hq + Hkv) * d
        table = min(case["axes"] * T, TABLE) * rot * 4 + 8 * case["axes"] * T
        if case["op"] == "rope":
            return {"bytes": 4 * elements + table, "flops": 10 * elements}
        written = T * Hkv * d * 17 // 16
        # queries and keys read, queries written, values read, codes written; then the codes read
        # and bf16 written
        return {"bytes": 2 * T * (2 * Hq + 2 * Hkv) * d + table + 8 * T + written
                + written + 4 * T * Hkv * d + 8 * T, "flops": 12 * elements}
    if case["op"] == "move":
        page = case["page"] * Hkv * d * 17 // 16
        return {"bytes": 2 * case["n"] * page * case["layers"] + 8 * case["n"], "flops": 0}
    lens, qs = _lens(case)
    w = case["window"]
    seen = sum(min(n, w + q - 1) if w else n for n, q in zip(lens, qs))
    return {"bytes": seen * Hkv * d * 17 // 16 + 4 * sum(qs) * Hq * d + 4 * (seen // case["page"]),
            "flops": 4 * d * Hq * sum(_pairs(n, q, w) for n, q in zip(lens, qs))}


# ---- the 4-bit format in plain torch ------------------------------------------------------------
def _halves(x):
    """Sum of the last axis, folded by halves."""
    n = x.shape[-1]
    return x[..., 0] if n == 1 else _halves(x[..., :n // 2] + x[..., n // 2:])


def _quantize(x):
    """fp32 [..., d] -> e2m1 codes [..., d] and scale bytes [..., d / 32], both uint8. The scale is
    the smallest power of two of which the block's largest magnitude is at most 7; a block with a
    value that is not finite is a block of NaN (255)."""
    b = x.unflatten(-1, (-1, 32))
    bits = b.abs().amax(-1).view(torch.int32)
    e = (((bits + 0x1FFFFF) >> 23) - 2).clamp(1, 254)
    e = torch.where(bits >= 0x7F800000, 255, e)
    a = b * ((254 - e).clamp(min=1) << 23).view(torch.float32)[..., None]
    m = a.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5)
            + (m >= 3.5) + (m > 5))
    return (code + 8 * torch.signbit(a).to(torch.uint8)).flatten(-2), e.to(torch.uint8)


@functools.lru_cache(maxsize=None)
def _e2m1(device):
    v = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float32, device=device)
    return torch.cat([v, -v])


def _values(codes, scales):
    """Codes [..., d] and scale bytes [..., d / 32] -> fp32 [..., d]."""
    e = scales.to(torch.int32)
    s = torch.where(e == 0, 0x400000, e << 23).view(torch.float32)
    s = torch.where(e == 255, torch.nan, s)
    v = _e2m1(codes.device)[codes.to(torch.int32)]
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _packed(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _value_shape(d):
    """(planes, bytes of a run): a value byte's place is [plane][token / 4][run][token % 4][byte]."""
    return (max(1, d // 128), 4 if d >= 128 else 2)


def _groups(k, v, d):
    """fp32 keys and values [..., 16, d] -> the bytes of their groups [..., 17 d]."""
    planes, run = _value_shape(d)
    kc, ks = _quantize(k)
    vc, vs = _quantize(v)
    vb = _packed(vc).unflatten(-2, (4, 4)).unflatten(-1, (planes, 16, run))
    n = vb.dim() - 5                    # [..., g, i, plane, r, byte] -> [..., plane, g, r, i, byte]
    vb = vb.permute(*range(n), n + 2, n, n + 3, n + 1, n + 4)
    return torch.cat([_packed(kc).flatten(-2), vb.flatten(-5), ks.flatten(-2),
                      vs.transpose(-1, -2).flatten(-2)], -1)


def _ungroups(b, d):
    """The bytes of groups [..., 17 d] -> fp32 keys and values [..., 16, d]."""
    planes, run = _value_shape(d)
    k = _values(_nibbles(b[..., :8 * d].unflatten(-1, (16, d // 2))),
                b[..., 16 * d:16 * d + d // 2].unflatten(-1, (16, d // 32)))
    vb = b[..., 8 * d:16 * d].unflatten(-1, (planes, 4, 16, 4, run))
    n = vb.dim() - 5
    vb = vb.permute(*range(n), n + 1, n + 3, n, n + 2, n + 4).flatten(-3).flatten(-3, -2)
    vs = b[..., 16 * d + d // 2:].unflatten(-1, (d // 32, 16)).transpose(-1, -2)
    return k, _values(_nibbles(vb), vs)


def _token_bytes(token, d):
    """Places in a group of the bytes of token 0..15: key codes, value codes, key scales, value
    scales."""
    planes, run = _value_shape(d)
    at = lambda n: torch.arange(n, device=token.device)  # noqa: E731
    t = token[..., None]
    plane, r, byte = at(planes)[:, None, None], at(16)[:, None], at(run)
    place = ((plane * 4) * 16 + r) * 4 * run + byte
    v = 8 * d + place.flatten() + ((t // 4) * 16 * 4 + t % 4) * run
    return torch.cat([t * (d // 2) + at(d // 2), v, 16 * d + t * (d // 32) + at(d // 32),
                      16 * d + d // 2 + at(d // 32) * 16 + t], -1)


# ---- inputs -------------------------------------------------------------------------------------
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _random_pages(g, pages, Hkv, page, d):
    """A cache of normalized keys and values."""
    n = pages * Hkv * (page // 16)
    out = torch.empty((n, 17 * d), dtype=torch.uint8, device="cuda")
    step = 1 << 17
    for at in range(0, n, step):
        m = min(step, n - at)
        out[at:at + m] = _groups(_normal(g, m, 16, d) * 1.2, _normal(g, m, 16, d), d)
    return out.view(pages, Hkv, page // 16, 17 * d)


def _sections(axes, half):
    return {1: [half], 2: [half // 2, half - half // 2],
            3: [half - 2 * (3 * half // 8), 3 * half // 8, 3 * half // 8]}[axes]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    Hq, Hkv, d, rot = HEADS[case["heads"]]
    s = dict(case=case)
    if case["op"] in ("rope", "append"):
        T, axes = case["T"], case["axes"]
        qkv = _normal(g, T, (Hq + 2 * Hkv) * d).to(torch.bfloat16)
        s["q"] = qkv[:, :Hq * d].unflatten(1, (Hq, d))
        s["k"] = qkv[:, Hq * d:(Hq + Hkv) * d].unflatten(1, (Hkv, d))
        s["v"] = qkv[:, (Hq + Hkv) * d:].unflatten(1, (Hkv, d))
        mean = 0.0 if case["gemma"] else 1.0
        s["qw"], s["kw"] = ((mean + 0.1 * _normal(g, d)).to(torch.bfloat16) for _ in range(2))
        inv = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
        angle = torch.arange(TABLE, dtype=torch.float64, device="cuda")[:, None] * inv
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).to(torch.float32)
        start = torch.randint(0, TABLE - T, (axes, 1), generator=g, device="cuda")
        s["pos"] = start + torch.arange(T, device="cuda")
        s["axis"] = None
        if axes == 1:
            s["pos"] = s["pos"][0]
        else:
            sec = torch.tensor(_sections(axes, rot // 2), device="cuda")
            s["axis"] = torch.repeat_interleave(torch.arange(axes, device="cuda"), sec).to(torch.int32)
        if case["op"] == "append":
            page = case["page"]
            pages = -(-2 * T // page) + 64
            s["cache"] = torch.randint(0, 120, (pages, Hkv, page // 16, 17 * d),
                                       dtype=torch.uint8, generator=g, device="cuda")
            if case["chunk"]:           # consecutive tokens through a list of pages
                table = torch.randperm(pages, generator=g, device="cuda")
                at = torch.arange(T, device="cuda") + page // 2 + 3
                s["slots"] = table[at // page] * page + at % page
            else:
                s["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:T].clone()
        return s
    if case["op"] == "move":
        layers, pages, n = case["layers"], case["pages"], case["n"]
        s["cache"] = torch.randint(0, 256, (layers, pages, Hkv, case["page"] // 16, 17 * d),
                                   dtype=torch.uint8, generator=g, device="cuda")
        order = torch.randperm(pages, generator=g, device="cuda")
        s["pairs"] = order[:2 * n].view(2, n).T.contiguous().to(torch.int32).cpu()
        s["tables"] = torch.randint(0, pages, (case["B"], 256), dtype=torch.int32, generator=g,
                                    device="cuda")
        return s
    lens, qs = _lens(case)
    page, B = case["page"], case["B"]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    s["cache"] = _random_pages(g, pages, Hkv, page, d)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((B, max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    s["pages"] = table
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    starts = [sum(qs[:b]) for b in range(B + 1)]
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["q"] = (_normal(g, starts[-1], Hq, d) * 1.5).to(torch.bfloat16)
    s["max_q"], s["max_len"] = max(qs), max(lens)
    return s


# ---- one pass -----------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _kv4():
    from vllm_sly_radiance_amd import radiance_kv4
    return radiance_kv4


def _norm_rope(x, w, s):
    """fp32 [T, heads, d]: the norm and the rotation, unrounded."""
    case = s["case"]
    T, H, d = x.shape
    half = HEADS[case["heads"]][3] // 2
    x = x.float()
    mean = _halves(_halves((x * x).unflatten(-1, (d // 8, 8)))) / d
    w = w.float() + 1.0 if case["gemma"] else w.float()
    y = x * (1.0 / torch.sqrt(mean + EPS))[..., None] * w
    pairs = torch.arange(half, device=x.device)
    pos = s["pos"][:, None] if s["axis"] is None else s["pos"][s["axis"].long()].T
    c, sn = s["table"][pos, pairs][:, None], s["table"][pos, pairs + half][:, None]
    lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["adjacent"] else \
        (slice(0, half), slice(half, 2 * half))
    out = y.clone()
    out[..., lo] = y[..., lo] * c - y[..., hi] * sn
    out[..., hi] = y[..., hi] * c + y[..., lo] * sn
    return out


def _plain_append(s):
    q = _norm_rope(s["q"], s["qw"], s).to(torch.bfloat16)
    k = _norm_rope(s["k"], s["kw"], s)
    (kc, ks), (vc, vs) = _quantize(k), _quantize(s["v"].float())
    cache = s["cache"]
    T, Hkv, d = k.shape
    page = cache.shape[2] * 16
    at = s["slots"] % page
    where = ((s["slots"] // page)[:, None, None], torch.arange(Hkv, device=k.device)[:, None],
             (at // 16)[:, None, None], _token_bytes(at % 16, d)[:, None])
    cache[where] = torch.cat([_packed(kc), _packed(vc), ks, vs], -1)
    b = cache[where]
    return q, _values(_nibbles(b[..., :d // 2]), b[..., d:d + d // 32]).to(torch.bfloat16), \
        _values(_nibbles(b[..., d // 2:d]), b[..., d + d // 32:]).to(torch.bfloat16)


def _plain_attention(s):
    case = s["case"]
    Hq, Hkv, d, _ = HEADS[case["heads"]]
    B, Q, L = case["B"], s["max_q"], s["max_len"]
    dev = s["q"].device
    k, v = _ungroups(s["cache"][s["pages"].long()], d)      # [B, pages, Hkv, groups, 16, d]
    k, v = (t.permute(0, 2, 1, 3, 4, 5).reshape(B, Hkv, -1, d)[:, :, :L] for t in (k, v))
    starts, lens = s["starts"].long(), s["lens"].long()
    n = starts[1:] - starts[:-1]
    i, j = torch.arange(Q, device=dev), torch.arange(L, device=dev)
    rows = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[rows].unflatten(2, (Hkv, Hq // Hkv)).permute(0, 2, 3, 1, 4)
    scores = (q.reshape(B, Hkv, -1, d) @ k.transpose(-1, -2)).view(B, Hkv, Hq // Hkv, Q, L)
    scores = scores * (1.0 / math.sqrt(d))
    last = (lens - n)[:, None] + i                          # each query's own place
    seen = (j <= last[..., None]) & (j < lens[:, None, None])
    if case["window"]:
        seen = seen & (j > last[..., None] - case["window"])
    scores = scores.masked_fill(~seen[:, None, None], -torch.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-3e38))
    o = (p.view(B, Hkv, -1, L) @ v).view(B, Hkv, -1, Q, d) / p.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, Q, Hq, d)
    return o[i < n[:, None]].to(torch.bfloat16)


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        K = _kv4()
        if op == "rope":
            return K.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["table"], s["pos"],
                                  axis=s["axis"], eps=EPS, plus_one=case["gemma"],
                                  adjacent=case["adjacent"])
        if op == "append":
            q = K.qk_norm_rope_append(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["table"],
                                      s["pos"], s["cache"], s["slots"], axis=s["axis"], eps=EPS,
                                      plus_one=case["gemma"], adjacent=case["adjacent"])
            return (q, *K.gather(s["cache"], s["slots"]))
        if op == "move":
            K.move_pages(s["cache"], s["pairs"], s["tables"])
            return s["cache"], s["tables"]
        return K.attention(s["q"], s["cache"], s["pages"], s["lens"], s["starts"], s["max_q"],
                           s["max_len"], window=case["window"])
    if op == "rope":
        return tuple(_norm_rope(s[x], s[x + "w"], s).to(torch.bfloat16) for x in "qk")
    if op == "append":
        return _plain_append(s)
    if op == "move":
        cache, tables = s["cache"], s["tables"]
        pairs = s["pairs"].to(cache.device).long()
        cache[:, pairs[:, 1]] = cache[:, pairs[:, 0]]
        new = torch.arange(case["pages"], dtype=torch.int32, device=cache.device)
        new[pairs[:, 0]] = pairs[:, 1].to(torch.int32)
        tables.copy_(new[tables.long()])
        return cache, tables
    return _plain_attention(s)


# ---- the definition in 64 bits ------------------------------------------------------------------
def _exact_rotated(x, w, s, case, rot):
    x = x.double()
    y = x / torch.sqrt(torch.mean(x ** 2, -1, keepdim=True) + EPS)
    y = y * (w.double() + (1 if case["gemma"] else 0))
    half = rot // 2
    z = torch.zeros((*x.shape[:2], half), dtype=torch.complex128, device=x.device)
    for p in range(half):
        a, b = (2 * p, 2 * p + 1) if case["adjacent"] else (p, p + half)
        pos = s["pos"] if s["axis"] is None else s["pos"][int(s["axis"][p])]
        turn = torch.complex(s["table"][pos, p].double(), s["table"][pos, half + p].double())
        z[..., p] = torch.complex(y[..., a], y[..., b]) * turn[:, None]
    out = y.clone()
    for p in range(half):
        a, b = (2 * p, 2 * p + 1) if case["adjacent"] else (p, p + half)
        out[..., a], out[..., b] = z[..., p].real, z[..., p].imag
    return out


def _exact_rounded(x):
    """float64 [..., d] -> the values that the 4-bit format holds for it."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 7))
    e = e + (torch.ldexp(torch.full_like(top, 7.0), e) < top).double()
    e = e - (torch.ldexp(torch.full_like(top, 7.0), e - 1) >= top).double()
    a = torch.ldexp(b, -e)
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    return torch.ldexp((torch.round(a / step) * step).clamp(-6, 6), e).reshape(x.shape)


def _exact_cached(groups, d):
    """Groups [n, 17 d] of consecutive tokens -> float64 keys and values [16 n, d]."""
    def value(c):
        c = c.long()
        e, m = (c >> 1) & 3, (c & 1).double()
        mag = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.double() - 1))
        return torch.where(c & 8 > 0, -mag, mag)
    n = groups.shape[0]
    planes, run = max(1, d // 128), 4 if d >= 128 else 2
    ks = groups[:, 16 * d:16 * d + d // 2].reshape(n * 16, d // 32)
    vs = groups[:, 16 * d + d // 2:].reshape(n, d // 32, 16).permute(0, 2, 1).reshape(n * 16, -1)
    kb = groups[:, :8 * d].reshape(n * 16, d // 2)
    vb = groups[:, 8 * d:16 * d].reshape(n, planes, 4, 16, 4, run)
    vb = torch.einsum("npgrib->ngiprb", vb.to(torch.int32)).reshape(n * 16, d // 2)
    out = []
    for b, e in ((kb, ks), (vb, vs)):
        x = torch.empty((n * 16, d), dtype=torch.float64, device=groups.device)
        x[:, 0::2], x[:, 1::2] = value(b % 16), value(b // 16)
        out.append(x * torch.exp2(e.double() - 127).repeat_interleave(32, dim=1))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    Hq, Hkv, d, rot = HEADS[case["heads"]]
    if case["op"] == "move":
        return None                     # bytes and page numbers
    if case["op"] in ("rope", "append"):
        q, k = (_exact_rotated(s[x], s[x + "w"], s, case, rot) for x in "qk")
        return (q, k) if case["op"] == "rope" else \
            (q, _exact_rounded(k), _exact_rounded(s["v"].double()))
    out = []
    lens, qs = _lens(case)
    at = 0
    for b, (n, m) in enumerate(zip(lens, qs)):
        pages = s["pages"][b, :-(-n // case["page"])].long()
        q = s["q"][at:at + m].double()
        at += m
        place = torch.arange(n - m, n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)
        hide = j > place
        if case["window"]:
            hide |= j <= place - case["window"]
        o = torch.empty((m, Hq, d), dtype=torch.float64, device=q.device)
        for h in range(Hkv):
            k, v = _exact_cached(s["cache"][pages, h].reshape(-1, 17 * d), d)
            for a in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                t = (q[:, a] @ k[:n].T) / math.sqrt(d)
                o[:, a] = torch.softmax(t.masked_fill(hide, -math.inf), -1) @ v[:n]
        out.append(o)
    return torch.cat(out)
