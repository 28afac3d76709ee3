"""CPU oracle of the attention operators over the 4-bit cache (numpy).

Two kinds of function: the steps whose bits are fixed (head norm, rotation, rounding to the cache's
format) restated in fp32 in the same order, and the definitions in float64.

A cache is uint8 [pages, heads, page / 16, 17 d]; 16 tokens of a head are key codes [16][d/2], value
codes [planes][4][16][4][bytes], key scales [16][d/32], value scales [d/32][16].
"""
from __future__ import annotations

import numpy as np

from .mxfp4_oracle import bf16_to_f32, f32_to_bf16

F32 = np.float32
E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])


# ---- the format ---------------------------------------------------------------------------------
def quantize(x: np.ndarray):
    """fp32 [..., d] -> (codes uint8 [..., d], scale bytes [..., d / 32])."""
    b = np.ascontiguousarray(x, F32).reshape(*x.shape[:-1], -1, 32)
    bits = (b.view(np.uint32) & 0x7FFFFFFF).max(-1)
    e = np.clip(((bits.astype(np.int64) + 0x1FFFFF) >> 23) - 2, 1, 252)
    nan = bits >= 0x7F800000
    with np.errstate(invalid="ignore", over="ignore"):
        a = b.astype(np.float64) * np.ldexp(1.0, 127 - e)[..., None]
        m = np.abs(a)
        c = ((m > 0.25).astype(np.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5)
             + (m >= 3.5) + (m > 5)).astype(np.uint8)
    c = c + 8 * np.signbit(b).astype(np.uint8)
    c[nan] = 0
    e[nan] = 255
    return c.reshape(x.shape), e.astype(np.uint8)


def dequantize(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """-> float64 [..., d]; a block of a scale above 252, the largest that quantize gives, is NaN."""
    s = np.ldexp(1.0, scales.astype(np.int64) - 127)
    s = np.where(scales > 252, np.nan, s)
    return E2M1[codes] * np.repeat(s, 32, axis=-1)


def _value_place(token: int, d: int) -> np.ndarray:
    """Byte places of the d / 2 value bytes of token 0..15 in its group."""
    planes, run = max(1, d // 128), 4 if d >= 128 else 2
    p, r, b = np.meshgrid(np.arange(planes), np.arange(16), np.arange(run), indexing="ij")
    return (8 * d + (((p * 4 + token // 4) * 16 + r) * 4 + token % 4) * run + b).reshape(-1)


def places(token: int, d: int):
    """(key codes, value codes, key scales, value scales) byte places of a token in its group."""
    n = d // 32
    return (token * (d // 2) + np.arange(d // 2), _value_place(token, d),
            16 * d + token * n + np.arange(n), 16 * d + d // 2 + np.arange(n) * 16 + token)


def write(cache: np.ndarray, slots, k: np.ndarray, v: np.ndarray) -> None:
    """Rounds fp32 k, v [T, heads, d] into the slots of the cache; slots outside it are skipped."""
    pages, H, groups, b = cache.shape
    d, page = b // 17, groups * 16
    pack = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)  # noqa: E731
    (kc, ks), (vc, vs) = quantize(k), quantize(v)
    for t, s in enumerate(np.asarray(slots, np.int64)):
        if s < 0 or s >= pages * page:
            continue
        pk, pv, sk, sv = places(int(s % 16), d)
        at = cache[s // page, :, (s % page) // 16]
        at[:, pk], at[:, pv], at[:, sk], at[:, sv] = pack(kc[t]), pack(vc[t]), ks[t], vs[t]


def read(cache: np.ndarray, slots):
    """float64 k, v [T, heads, d] of the slots; zeros below 0, NaN past the end."""
    pages, H, groups, b = cache.shape
    d, page = b // 17, groups * 16
    nib = lambda x: np.stack([x & 15, x >> 4], -1).reshape(*x.shape[:-1], -1)  # noqa: E731
    k = np.zeros((len(slots), H, d))
    v = np.zeros((len(slots), H, d))
    for t, s in enumerate(np.asarray(slots, np.int64)):
        if s < 0:
            continue
        if s >= pages * page:
            k[t], v[t] = np.nan, np.nan
            continue
        pk, pv, sk, sv = places(int(s % 16), d)
        at = cache[s // page, :, (s % page) // 16]
        k[t] = dequantize(nib(at[:, pk]), at[:, sk])
        v[t] = dequantize(nib(at[:, pv]), at[:, sv])
    return k, v


# ---- head norm and rotation ---------------------------------------------------------------------
def _halves(x: np.ndarray) -> np.ndarray:
    while x.shape[-1] > 1:
        n = x.shape[-1] // 2
        x = x[..., :n] + x[..., n:]
    return x[..., 0]


def _turns(table, positions, axis, T, dtype):
    """cos, sin [T, rot / 2] (NaN where a position or axis is out of range)."""
    rows, rot = table.shape
    half = rot // 2
    pos = np.atleast_2d(np.asarray(positions))
    axis = np.zeros(half, np.int64) if axis is None else np.asarray(axis)
    c = np.full((T, half), np.nan, dtype)
    s = np.full((T, half), np.nan, dtype)
    for p in range(half):
        if not 0 <= axis[p] < pos.shape[0]:
            continue
        at = pos[axis[p]]
        ok = (at >= 0) & (at < rows)
        c[ok, p], s[ok, p] = table[at[ok], p], table[at[ok], half + p]
    return c, s


def norm_rope(x_bits, w_bits, table, positions, axis=None, eps=1e-6, plus_one=False, adjacent=False,
              dtype=F32):
    """bf16 bits x [T, H, d], weight bits [d] or None, table [rows, rot] (or None) -> unrounded
    [T, H, d] in dtype: float32 follows the kernel's steps bit for bit, float64 is the definition."""
    x = bf16_to_f32(x_bits).astype(dtype)
    T, H, d = x.shape
    one = dtype(1.0)
    with np.errstate(all="ignore"):
        y = x
        if w_bits is not None:
            w = bf16_to_f32(w_bits).astype(dtype)
            w = w + one if plus_one else w
            sq = (x * x).reshape(T, H, d // 8, 8)
            mean = _halves(_halves(sq)) * dtype(1.0 / d)
            y = x * (one / np.sqrt(mean + dtype(F32(eps))))[..., None] * w
        if table is None:
            return y
        rot = table.shape[1]
        c, s = _turns(table.astype(dtype), positions, axis, T, dtype)
        c, s = c[:, None], s[:, None]
        half = rot // 2
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if adjacent else (slice(0, half),
                                                                     slice(half, rot))
        out = y.copy()
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
    return out


# ---- attention ----------------------------------------------------------------------------------
def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float, causal=True, window=0):
    """float64 q [n, Hq, d] of the last n of L tokens, k, v [L, Hkv, d] -> (o [n, Hq, d], the weighted
    |v| [n, Hq, d], the largest sum of |q_c k_c| * scale over a row's visible tokens [n, Hq]).
    Tokens that a row does not see do not enter it, whatever they hold."""
    n, Hq, d = q.shape
    L, Hkv = k.shape[0], k.shape[1]
    o, weight, terms = np.zeros((n, Hq, d)), np.zeros((n, Hq, d)), np.zeros((n, Hq))
    j = np.arange(L)
    for i in range(n):
        place = L - n + i
        see = (j <= place) if causal else j >= 0
        if window:
            see = see & (j > place - window)
        if not see.any():
            continue
        for h in range(Hq):
            kk, vv = k[see, h // (Hq // Hkv)], v[see, h // (Hq // Hkv)]
            s = kk @ q[i, h] * scale
            p = np.exp(s - s.max())
            p = p / p.sum()
            o[i, h], weight[i, h] = p @ vv, p @ np.abs(vv)
            terms[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * scale
    return o, weight, terms


def attention_tolerance(o, weight, terms, d):
    """Elementwise bound on a bf16 output whose weights are rounded to bf16 (round to nearest is off by
    at most 2^-8 of the value) and whose scores are fp32 sums of d products:
      output rounding   2^-8 |o|
      weight rounding   2^-8 sum p |v| (the normalizing sum is of the unrounded weights)
      score error       each weight off by a factor e^(+-x), x = (d + 2) 2^-24 terms, in the numerator
                        and in the normalizing sum, and 2^-18 for the fp32 sums and powers of two"""
    x = 2 * (d + 2) * 2.0 ** -24 * terms[..., None] + 2.0 ** -18
    return 2.0 ** -8 * np.abs(o) + (2.0 ** -8 + x) * 1.01 * weight + 1e-30
