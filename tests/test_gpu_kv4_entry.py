"""The ops of the 4-bit cache under torch.func.vmap, as tensor subclasses' arguments and from several Python
threads: the same results as called one by one."""
import threading

import numpy as np
import pytest
import torch

from tests._check import host_u16
from tests._kv4 import Batch
from vllm_sly_radiance_amd import _native_kv4
from vllm_sly_radiance_amd import radiance_kv4 as K

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_kv4.lib()


def test_vmap_is_the_loop():
    b = Batch(np.random.default_rng(1), [200, 33], [3, 1], 4, 2, 128, 16)
    q, cache, table, lens, starts, mq, ml = b.device()
    qs = torch.stack([q, q * 0.5, -q])
    ls = torch.stack([lens, lens - 5, lens - 20])
    got = torch.func.vmap(lambda q, n: K.attention(q, cache, table, n, starts, mq, ml))(qs, ls)
    for i in range(3):
        assert torch.equal(got[i], K.attention(qs[i], cache, table, ls[i], starts, mq, ml))
    slots = torch.randint(0, 100, (4, 7), device="cuda")
    k, v = torch.func.vmap(lambda s: K.gather(cache, s))(slots)
    for i in range(4):
        wk, wv = K.gather(cache, slots[i])
        assert torch.equal(k[i], wk) and torch.equal(v[i], wv)


def test_threads_on_streams_of_their_own():
    batches = [Batch(np.random.default_rng(i), [900 + 700 * i, 40, 300], [1, 2, 1 + i], 8, 2, 128, 16)
               for i in range(4)]
    args = [b.device() for b in batches]
    want = [host_u16(K.attention(*a)) for a in args]
    torch.cuda.synchronize()
    wrong, outs = [], [None] * 4

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                outs[i] = [K.attention(*args[i]) for _ in range(30)]
                with pytest.raises(RuntimeError, match=f"max_len=-{i + 1}"):    # errors are a thread's own
                    K.attention(*args[i][:6], -(i + 1))
            stream.synchronize()
        except BaseException as e:  # noqa: BLE001
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for i in range(4):
        for o in outs[i]:
            assert np.array_equal(host_u16(o), want[i])
