"""Queries that are not finite, against the definition: an infinite one has only infinite or undefined scores,
so that its output is NaN like a NaN one's (zeros where it sees nothing), and the rows beside them in a workgroup
are not touched."""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as KO
from tests._kv4 import Batch
from vllm_sly_radiance_amd import _native_kv4
from vllm_sly_radiance_amd import radiance_kv4 as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_kv4.lib()


# (query heads, kv heads, d, page, lengths, queries): few rows, shared runs and their join, many rows, parts
SHAPES = [(4, 2, 128, 16, [37, 1, 15, 190], [1, 1, 4, 100]), (8, 2, 64, 16, [9, 131], [9, 9]),
          (6, 1, 256, 16, [77, 3], [5, 3]), (8, 2, 128, 16, [2300, 1777, 2], [1, 3, 2]),
          (8, 2, 256, 16, [2300, 4], [2, 4]), (64, 4, 128, 64, [417, 333], [400, 333]),
          (64, 2, 256, 32, [201, 230], [201, 200]), (32, 2, 128, 32, [1100], [401])]
INF, NAN = 0x7F80, 0x7FC0


def attend(b, **kw):
    q, cache, table, lens, starts, mq, ml = b.device()
    print(f"[kv4] lens={b.lens} q={b.qs} heads={q.shape[1]}/{b.Hkv} d={b.d} page={b.page} {kw}", flush=True)
    out = K.attention(q, cache, table, lens, starts, mq, ml, **kw)
    torch.cuda.synchronize()
    return out


def check(b, out, **kw):
    """NaN in the rows of queries that are not finite and see something; the bound for the others."""
    clean = (b.q & INF) != INF
    rows = clean.all(-1)
    saw = np.zeros(rows.shape, bool)
    for s, n in enumerate(b.lens):
        first = b.starts[s + 1] - n if kw.get("causal", True) else 0
        saw[b.starts[s]:b.starts[s + 1]] = (np.arange(b.starts[s], b.starts[s + 1]) >= first)[:, None] & (n > 0)
    got = out.float().cpu().numpy()
    assert np.isnan(got[~rows & saw]).all() and not got[~saw].any()
    # the others against the definition, with queries of zero (which no row shares) in the place of these
    whole, b.q = b.q, np.where(rows[..., None], b.q, 0).astype(np.uint16)
    fixed = attend(b, **kw)
    b.check(torch.where(torch.from_numpy(rows).cuda()[..., None], out, fixed), **kw)
    b.q = whole


@pytest.mark.parametrize("window", [0, 3])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_one_channel_not_finite(shape, window):
    Hq, Hkv, d, page, lens, qs = SHAPES[shape]
    rng = np.random.default_rng(shape)
    b = Batch(rng, lens, qs, Hq, Hkv, d, page)
    for i in range(b.q.shape[0]):
        for h in range(Hq):
            what = rng.integers(8)
            if what < 3:
                b.q[i, h, rng.integers(d)] = (INF, 0x8000 | INF, NAN)[what]
    check(b, attend(b, window=window), window=window)


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_every_score_infinite(shape):
    """All keys 1: a query of -infinity has only scores of -infinity, whose weights are 0 / 0 and not nothing;
    one with a single such channel likewise."""
    Hq, Hkv, d, page, lens, qs = SHAPES[shape]
    b = Batch(np.random.default_rng(shape), lens, qs, Hq, Hkv, d, page)
    for t in range(16):
        pk, _, sk, _ = KO.places(t, d)
        b.cache[..., pk], b.cache[..., sk] = 0x22, 127
    b.q[::2, 0] = 0x8000 | INF
    b.q[1::3, Hq - 1, 5] = 0x8000 | INF
    b.q[::5, Hq // 2] = INF
    check(b, attend(b))
    check(b, attend(b, window=20, causal=False), window=20, causal=False)
