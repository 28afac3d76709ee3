"""Shared helpers of the tests of the 4-bit cache and its attention."""
import numpy as np
import torch

from oracle import kv4_oracle as KO
from oracle import mxfp4_oracle as O
from tests._check import bf16_dev, host_u16, to_dev


def bits(rng, *shape, scale=1.0, mean=0.0):
    return O.f32_to_bf16((mean + scale * rng.standard_normal(shape)).astype(np.float32))


def random_cache(rng, pages, heads, page, d):
    """A cache of rounded normal keys and values."""
    cache = np.zeros((pages, heads, page // 16, 17 * d), np.uint8)
    slots = np.arange(pages * page)
    k = rng.standard_normal((len(slots), heads, d)).astype(np.float32)
    v = rng.standard_normal((len(slots), heads, d)).astype(np.float32)
    KO.write(cache, slots, k, v)
    return cache


def angles(rows, rot, base=1e4):
    a = np.arange(rows)[:, None] * base ** (-np.arange(0, rot, 2) / rot)
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


class Batch:
    """Sequences of a cache: their pages in a shuffled order, the page table and the oracle's view."""

    def __init__(self, rng, lens, qs, Hq, Hkv, d, page, extra=2, q_scale=1.5):
        self.lens, self.qs, self.page, self.d, self.Hkv = lens, qs, page, d, Hkv
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + extra
        self.cache = random_cache(rng, self.pages, Hkv, page, d)
        order = rng.permutation(self.pages)
        self.table = np.full((len(lens), max(max(need, default=0), 1)), -7, np.int32)
        at = 0
        for b, m in enumerate(need):
            self.table[b, :m] = order[at:at + m]
            at += m
        self.spare = order[at:]
        self.starts = np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)
        self.q = bits(rng, int(self.starts[-1]), Hq, d, scale=q_scale)

    def slots(self, b):
        t = np.arange(self.lens[b])
        return self.table[b][t // self.page].astype(np.int64) * self.page + t % self.page

    def device(self):
        i32 = lambda a: to_dev(np.asarray(a, np.int32))  # noqa: E731
        return (bf16_dev(self.q), to_dev(self.cache), i32(self.table), i32(self.lens),
                i32(self.starts), max(self.qs), max(self.lens))

    def check(self, out, scale=None, causal=True, window=0, only=None):
        """out bf16 [total, Hq, d] against the definition; returns the worst error over its bound."""
        got = O.bf16_to_f32(host_u16(out)).astype(np.float64)
        scale = 1 / np.sqrt(self.d) if scale is None else scale
        worst = 0.0
        for b in range(len(self.lens)):
            if only is not None and b not in only:
                continue
            a, e = self.starts[b], self.starts[b + 1]
            k, v = KO.read(self.cache, self.slots(b))
            q = O.bf16_to_f32(self.q[a:e]).astype(np.float64)
            with np.errstate(invalid="ignore"):
                o, w, t = KO.attention(q, k, v, scale, causal, window)
                tol = KO.attention_tolerance(o, w, t, self.d)
            g = got[a:e]
            assert np.array_equal(np.isnan(g), np.isnan(o)), \
                f"sequence {b}: NaN at {np.argwhere(np.isnan(g) != np.isnan(o))[:4].tolist()}"
            fin = ~np.isnan(o)
            if fin.any():
                worst = max(worst, float((np.abs(g - o)[fin] / tol[fin]).max()))
        assert worst <= 1.0, f"{worst:.3g} times the bound"
        return worst
