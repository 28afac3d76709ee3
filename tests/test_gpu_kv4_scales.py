"""Scale bytes of the 4-bit cache that append never writes. 252 is the largest it does (6 x 2^125 is the
largest of its values that bf16 holds); those above read as NaN, as 255 does, and like it only to the
queries that see the token."""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as KO
from oracle import mxfp4_oracle as O
from tests._check import host_u16, to_dev
from tests._kv4 import Batch
from vllm_sly_radiance_amd import _native_kv4
from vllm_sly_radiance_amd import radiance_kv4 as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_kv4.lib()


def attend(b, **kw):
    q, cache, table, lens, starts, mq, ml = b.device()
    print(f"[kv4] lens={b.lens} q={b.qs} heads={q.shape[1]}/{b.Hkv} d={b.d} page={b.page} {kw}", flush=True)
    out = K.attention(q, cache, table, lens, starts, mq, ml, **kw)
    torch.cuda.synchronize()
    return out


# (query heads, kv heads, d, page, lengths, queries): few rows, shared runs, many rows
SHAPES = [(4, 2, 128, 32, [37, 1, 15, 190], [1, 1, 4, 100]), (4, 2, 64, 16, [50, 131], [1, 9]),
          (6, 1, 256, 16, [77, 40], [5, 2]), (8, 2, 128, 16, [2300, 1777], [1, 3]),
          (64, 4, 128, 64, [417, 333, 30], [400, 320, 1]), (64, 4, 64, 16, [401, 350], [390, 350]),
          (64, 2, 256, 32, [270, 201], [200, 200])]


@pytest.mark.parametrize("scale,code", [(253, 0x77), (253, 0xFF), (254, 0x77), (254, 0xFF), (254, 0x27)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_what_lies_behind_the_sequence_has_no_effect(shape, scale, code):
    Hq, Hkv, d, page, lens, qs = SHAPES[shape]
    b = Batch(np.random.default_rng(shape), lens, qs, Hq, Hkv, d, page)
    want = host_u16(attend(b))
    used = np.zeros((b.pages, b.page), bool)
    for s in range(len(b.lens)):
        used.reshape(-1)[b.slots(s)] = True
    for p, t in np.argwhere(~used):
        pk, pv, sk, sv = KO.places(int(t % 16), d)
        for part, fill in ((pk, code), (pv, code), (sk, scale), (sv, scale)):
            b.cache[p, :, t // 16, part] = fill
    assert np.array_equal(host_u16(attend(b)), want)


@pytest.mark.parametrize("window", [0, 35])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_they_reach_the_queries_that_see_them(shape, window):
    Hq, Hkv, d, page, lens, qs = SHAPES[shape]
    rng = np.random.default_rng(shape)
    b = Batch(rng, lens, qs, Hq, Hkv, d, page)
    for s, n in enumerate(lens):
        for tok, head, what, scale in ((n - 1, 0, 3, 253), (n // 2, Hkv - 1, 3, 254), (n // 3, 0, 2, 253),
                                       (n - n // 4 - 1, Hkv - 1, 2, 254), (0, 0, 3, 254)):
            slot = b.slots(s)[tok]
            places = KO.places(int(slot % 16), d)
            at = b.cache[slot // page, head, (slot % page) // 16]
            at[places[what][int(rng.integers(d // 32))]] = scale
    b.check(attend(b, window=window), window=window)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_gather(d):
    rng = np.random.default_rng(d)
    cache = rng.integers(0, 256, (3, 2, 2, 17 * d), dtype=np.uint8)
    cache[..., 16 * d:] = rng.integers(250, 256, (3, 2, 2, d), dtype=np.uint8)
    slots = np.arange(96)
    for got, want in zip(K.gather(to_dev(cache), to_dev(slots)), KO.read(cache, slots)):
        assert 0.3 < np.isnan(want).mean() < 0.7
        assert np.array_equal(O.bf16_to_f32(host_u16(got)).astype(np.float64), want, equal_nan=True)
