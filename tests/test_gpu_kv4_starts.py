"""Query starts that the launch of an attention over the 4-bit cache was not sized for: the kernels stay in
their buffers, and the calls after are right. Starts of a batch that is padded to one size."""
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


@pytest.mark.parametrize("d,Hq,Hkv,q,n", [(128, 64, 8, 400, 63), (64, 64, 64, 300, 9), (256, 32, 4, 300, 31),
                                          (128, 8, 2, 3, 63)])
def test_starts_that_go_back(d, Hq, Hkv, q, n):
    """The same rows over and over: many more row tiles than the rows in all would make."""
    b = Batch(np.random.default_rng(n), [q + 900], [q], Hq, Hkv, d, 16)
    rows, cache, table, _, starts, _, ml = b.device()
    lens = torch.full((n,), ml, dtype=torch.int32, device="cuda")
    back = torch.tensor([0, q] * ((n + 1) // 2), dtype=torch.int32, device="cuda")
    print(f"[kv4] starts that go back d={d} heads={Hq}/{Hkv} {n} x {q} queries", flush=True)
    out = K.attention(rows, cache, table.expand(n, -1), lens, back, q, ml)
    torch.cuda.synchronize()
    assert out.shape == rows.shape
    b.check(K.attention(rows, cache, table, lens[:1], starts, q, ml))


@pytest.mark.parametrize("d,Hq,Hkv,qs", [(128, 64, 8, [300, 10, 190, 1]), (64, 32, 4, [290, 0, 290]),
                                         (256, 16, 2, [280, 270, 33]), (128, 8, 2, [4, 1, 2, 3]),
                                         (128, 32, 8, [1, 0, 1, 1])])
def test_a_batch_padded_to_one_size(d, Hq, Hkv, qs):
    """As many rows as max_q times the batch, of which the sequences own fewer."""
    most = max(qs)
    rng = np.random.default_rng(d)
    for extra in (40, 1500):
        b = Batch(rng, [n + extra - i for i, n in enumerate(qs)], qs, Hq, Hkv, d, 16)
        q, cache, table, lens, starts, mq, ml = b.device()
        padded = torch.full((len(qs) * most, Hq, d), 7.0, dtype=torch.bfloat16, device="cuda")
        padded[:q.shape[0]] = q
        print(f"[kv4] padded d={d} heads={Hq}/{Hkv} q={qs} + {extra}", flush=True)
        b.check(K.attention(padded, cache, table, lens, starts, mq, ml)[:q.shape[0]])
