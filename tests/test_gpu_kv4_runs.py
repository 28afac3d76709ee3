"""GPU parity of the attention over the 4-bit cache where the cached tokens of a batch are shared out over
workgroups: few rows against long contexts, among short ones, within the bound that
oracle.kv4_oracle.attention_tolerance derives."""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as KO
from oracle import mxfp4_oracle as O
from tests._check import host_u16
from tests._kv4 import Batch
from vllm_sly_radiance_amd import _native_kv4
from vllm_sly_radiance_amd import radiance_kv4 as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_kv4.lib()


def run(batch, **kw):
    q, cache, table, lens, starts, mq, ml = batch.device()
    # shared out, which takes a workspace (tests/test_kv4_abi_cpu.py has the rule)
    assert _native_kv4.attention_workspace(q.shape[0], len(batch.lens), mq, ml, q.shape[1], batch.Hkv,
                                           batch.d, kw.get("window", 0)) > 0
    print(f"[kv4] lens={batch.lens[:8]} q={batch.qs[:8]} heads={q.shape[1]}/{batch.Hkv} d={batch.d} "
          f"page={batch.page} {kw}", flush=True)
    out = K.attention(q, cache, table, lens, starts, mq, ml, **kw)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("d,page", [(64, 16), (128, 32), (256, 64)])
@pytest.mark.parametrize("Hq,Hkv,q", [(4, 4, 1), (8, 2, 1), (8, 2, 4), (6, 2, 9), (8, 1, 7)])
@pytest.mark.parametrize("window,causal", [(0, True), (0, False), (2500, True)])
def test_long_among_short(d, page, Hq, Hkv, q, window, causal):
    """Long contexts, one token, none, and lengths about a granule; one, two and four fragments of rows."""
    lens = [3001, 1, 0, 127, 2600, 129, 128, 1500]
    qs = [q, 1, 0, min(q, 2), q, q, 1, q]
    b = Batch(np.random.default_rng(1), lens, qs, Hq, Hkv, d, page)
    b.check(run(b, window=window, causal=causal), window=window, causal=causal)


@pytest.mark.parametrize("lens", [[4096] * 4, [4224], [2048, 4096, 1024], [4500] + [60] * 90])
def test_whole_runs_and_more_units_than_runs(lens):
    """Units that are whole numbers of runs, and more units than there are runs."""
    b = Batch(np.random.default_rng(2), lens, [1] * len(lens), 16, 16, 64, 16)
    b.check(run(b))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q", [1, 5, 17])
def test_nan_blocks_far_into_a_context(d, q):
    lens = [2200, 40, 1900]
    b = Batch(np.random.default_rng(3), lens, [q, 1, q], 8, 2, d, 16)
    for s, tok, head, what in ((0, 5, 0, "v"), (0, 2195, 0, "v"), (0, 1000, 1, "k"), (1, 39, 1, "v"),
                               (2, 1899, 0, "v"), (2, 1895, 0, "k")):
        slot = b.slots(s)[tok]
        pk, pv, sk, sv = KO.places(int(slot % 16), d)
        b.cache[slot // 16, head, 0][(sk if what == "k" else sv)[tok % (d // 32)]] = 255
    b.check(run(b))


def test_bad_pages_and_lengths_far_into_a_context():
    b = Batch(np.random.default_rng(4), [2500, 1800, 60, 1700], [2, 1, 1, 3], 8, 2, 128, 16)
    page = b.table[0, 100]
    b.table[0, 100] = b.pages
    out = run(b)
    assert np.isnan(O.bf16_to_f32(host_u16(out))[:2]).all()
    b.check(out, only=(1, 2, 3))
    b.table[0, 100] = page
    q, cache, table, lens, starts, mq, ml = b.device()
    wrong = lens.clone()
    wrong[1] = -1
    wrong[3] = 2501
    out = K.attention(q, cache, table, wrong, starts, mq, ml)
    got = O.bf16_to_f32(host_u16(out))
    assert np.isnan(got[2]).all() and np.isnan(got[4:]).all()
    b.check(out, only=(0, 2))


def test_graph_serves_lengths_that_share_out_otherwise():
    """One captured launch: replays with other lengths find other runs."""
    rng = np.random.default_rng(5)
    batches = [Batch(rng, n, [1] * 5, 8, 2, 128, 16)
               for n in ([3000, 10, 500, 2999, 0], [1, 1, 1, 1, 1], [0] * 5, [3000] * 5, [700, 3000, 3, 90, 2048])]
    pages = max(x.pages for x in batches)
    q = torch.zeros((5, 8, 128), dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros((pages, *batches[0].cache.shape[1:]), dtype=torch.uint8, device="cuda")
    table = torch.zeros((5, 188), dtype=torch.int32, device="cuda")
    lens = torch.zeros(5, dtype=torch.int32, device="cuda")
    starts = torch.arange(6, dtype=torch.int32, device="cuda")

    def load(x):
        dq, dc, dt, dl, _, _, _ = x.device()
        q.copy_(dq)
        cache[:dc.shape[0]] = dc
        table[:, :dt.shape[1]] = dt
        lens.copy_(dl)
        torch.cuda.synchronize()

    load(batches[0])
    K.attention(q, cache, table, lens, starts, 1, 3000)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            out = K.attention(q, cache, table, lens, starts, 1, 3000)
    for i in (3, 0, 1, 4, 2, 0):
        load(batches[i])
        g.replay()
        torch.cuda.synchronize()
        batches[i].check(out)
        assert torch.equal(out, K.attention(q, cache, table, lens, starts, 1, 3000))
