"""Attention over the 4-bit cache under limits far above what a batch holds."""
import numpy as np
import pytest
import torch

from tests._kv4 import Batch
from vllm_sly_radiance_amd import _native_kv4
from vllm_sly_radiance_amd import radiance_kv4 as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_kv4.lib()


@pytest.mark.parametrize("Hq,Hkv,d,n,chunk,max_q", [(32, 8, 128, 512, 150, 4096), (48, 16, 128, 256, 70, 4096),
                                                    (16, 2, 256, 300, 1, 8192)])
def test_a_chunk_beside_many_decoding_sequences(Hq, Hkv, d, n, chunk, max_q):
    """Limits of 131072 tokens and thousands of queries a sequence, as of a server's captured graph."""
    rng = np.random.default_rng(n)
    qs = [1] * n
    qs[n // 3] = chunk
    lens = [int(x) for x in rng.integers(1, 40, n)]
    lens[n // 3] = chunk + 60
    b = Batch(rng, lens, qs, Hq, Hkv, d, 16)
    q, cache, table, dl, starts, _, _ = b.device()
    rows = torch.zeros((n - 1 + max_q, Hq, d), dtype=torch.bfloat16, device="cuda")
    rows[:q.shape[0]] = q
    wide = torch.full((n, 131072 // 16), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    print(f"[kv4] {n} sequences, heads={Hq}/{Hkv} d={d} chunk {chunk} of {max_q}", flush=True)
    b.check(K.attention(rows, cache, wide, dl, starts, max_q, 131072)[:q.shape[0]])


@pytest.mark.parametrize("max_len", [30, 100000])
@pytest.mark.parametrize("d,qs", [(128, [2, 0, 1]), (64, [300, 1, 200]), (256, [0, 0, 0])])
def test_no_queries_allowed(d, qs, max_len):
    """max_q = 0: every sequence with queries has more than that, and its rows are NaN as under any max_q."""
    cache = K.new_cache(4, 2, 16, d)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.ones((sum(qs) + 3, 8, d), dtype=torch.bfloat16, device="cuda")
    table = torch.zeros((3, 7000), dtype=torch.int32, device="cuda")
    starts = i32(0, qs[0], qs[0] + qs[1], sum(qs))
    print(f"[kv4] max_q=0 q={qs} d={d} max_len={max_len}", flush=True)
    for lens in (i32(30, 20, 25), i32(0, 0, 0)):
        assert K.attention(q, cache, table, lens, starts, 0, max_len)[:sum(qs)].isnan().all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 8, 1 << 20, 130])
@pytest.mark.parametrize("d,Hq,Hkv,lens,qs", [(128, 4, 2, [5, 0, 20], [9, 3, 1]), (64, 4, 2, [2500, 7], [1, 30]),
                                              (128, 64, 8, [120, 130], [250, 130])])
def test_windows_longer_than_any_sequence(d, Hq, Hkv, lens, qs, window, causal):
    """As large as an int: queries that stand before the sequence (more of them than tokens) reach far below
    zero."""
    b = Batch(np.random.default_rng(d), lens, qs, Hq, Hkv, d, 16)
    q, cache, table, dl, starts, mq, ml = b.device()
    print(f"[kv4] lens={lens} q={qs} d={d} window={window} causal={causal}", flush=True)
    out = K.attention(q, cache, table, dl, starts, mq, ml, causal=causal, window=window)
    b.check(out, causal=causal, window=window)
