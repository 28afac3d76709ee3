"""Attention over the 4-bit cache where pages cannot be read: caches of no pages, page numbers outside the
cache. What a query does not see has no effect on it."""
import numpy as np
import pytest
import torch

from tests._check import host_u16, to_dev
from tests._kv4 import Batch
from vllm_sly_radiance_amd import _native_kv4
from vllm_sly_radiance_amd import radiance_kv4 as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_kv4.lib()


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# few rows in a workgroup a unit, in shared runs with the join, many rows, and both kinds beside
@pytest.mark.parametrize("d,Hq,Hkv,qs,max_len", [(128, 4, 2, [1, 2], 60), (64, 4, 2, [1, 2], 5000),
                                                 (128, 64, 8, [300, 280], 400), (256, 32, 4, [300, 290], 400),
                                                 (128, 64, 8, [1, 400], 3000)])
@pytest.mark.parametrize("pages_of", [0, 7, -1])
def test_a_cache_of_no_pages(d, Hq, Hkv, qs, max_len, pages_of):
    """A sequence with tokens is NaN, whatever its page numbers; one without sees nothing."""
    cache = K.new_cache(0, Hkv, 16, d)
    q = torch.ones((sum(qs), Hq, d), dtype=torch.bfloat16, device="cuda")
    table = torch.full((2, 320), pages_of, dtype=torch.int32, device="cuda")
    for lens in ([0, max_len], [max_len, 0], [0, 0]):
        print(f"[kv4] no pages d={d} heads={Hq}/{Hkv} q={qs} lens={lens}", flush=True)
        out = K.attention(q, cache, table, i32(*lens), i32(0, qs[0], sum(qs)), max(qs), max_len)
        for n, rows in zip(lens, out.float().split(qs)):
            assert rows.isnan().all() if n else not rows.any()
    k, v = K.gather(cache, torch.tensor([0, 5, -1], device="cuda"))
    for x in (k, v):
        assert x[:2].isnan().all() and not x[2].any()


def attend(b, table, **kw):
    q, cache, _, lens, starts, mq, ml = b.device()
    print(f"[kv4] lens={b.lens} q={b.qs} heads={q.shape[1]}/{b.Hkv} d={b.d} page={b.page} {kw}", flush=True)
    out = K.attention(q, cache, to_dev(table), lens, starts, mq, ml, **kw)
    torch.cuda.synchronize()
    return out


# (query heads, kv heads, d, page, lengths, queries): decode, drafts, shared runs, chunks, both beside
SHAPES = [(4, 2, 128, 16, [116, 47, 300], [1, 1, 1]), (8, 2, 64, 16, [116, 90, 31], [4, 9, 2]),
          (4, 1, 256, 16, [215, 130], [1, 30]), (8, 2, 128, 16, [3000, 2517, 40], [1, 3, 1]),
          (8, 2, 64, 32, [2600, 1999], [5, 1]), (64, 8, 128, 16, [417, 390], [250, 210]),
          (64, 8, 64, 16, [333, 411], [222, 240]), (32, 4, 256, 16, [300, 260], [250, 200]),
          (64, 8, 128, 16, [500, 60, 77], [300, 1, 1]), (32, 2, 128, 32, [1300], [401])]


@pytest.mark.parametrize("window", [1, 17, 100, 115])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_pages_released_behind_a_window(shape, window):
    """The pages that lie wholly before what a sequence's first query sees belong to nobody any more."""
    Hq, Hkv, d, page, lens, qs = SHAPES[shape]
    b = Batch(np.random.default_rng(shape), lens, qs, Hq, Hkv, d, page)
    want = attend(b, b.table, window=window)
    b.check(want, window=window)
    for number in (-1, 1 << 30):
        table = b.table.copy()
        for i, (n, q) in enumerate(zip(lens, qs)):
            table[i, :max(n - q - window + 1, 0) // page] = number
        assert window > 17 or (table != b.table).any()
        assert np.array_equal(host_u16(attend(b, table, window=window)), host_u16(want))


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 50), (False, 0), (False, 90)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_unusable_pages_reach_the_queries_that_read_them(shape, causal, window):
    """Exactly those: not the ones before the page or past their window, in the same workgroup or not."""
    Hq, Hkv, d, page, lens, qs = SHAPES[shape]
    b = Batch(np.random.default_rng(shape), lens, qs, Hq, Hkv, d, page)
    table = b.table.copy()
    for i, (n, q) in enumerate(zip(lens, qs)):
        for tok in (n - 1 - q // 2, n - q - 40):
            if tok >= 0 and i != 1:
                # to the oracle, keys that are NaN
                at = tok // page
                b.cache[b.table[i, at], :, :, 16 * d:16 * d + d // 2] = 255
                table[i, at] = (b.pages, -1)[tok & 1]
    clean = b.cache.copy()
    clean[..., 16 * d:16 * d + d // 2] = np.minimum(clean[..., 16 * d:16 * d + d // 2], 130)
    marked, b.cache = b.cache, clean
    out = attend(b, table, causal=causal, window=window)
    b.cache = marked
    b.check(out, causal=causal, window=window)
