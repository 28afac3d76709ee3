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


def test_writes_into_the_cache_are_seen_by_autograd():
    """A tensor saved for a backward pass and written since is noticed, as after any op in place."""
    bf = lambda *s: torch.ones(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    slots = torch.arange(3, device="cuda")
    for write in (lambda c, t: K.qk_norm_rope_append(bf(3, 4, 64), bf(3, 2, 64), bf(3, 2, 64), None, None, None,
                                                     None, c, slots),
                  lambda c, t: K.move_pages(c, torch.tensor([[0, 1]], dtype=torch.int32), t)):
        for mode in (torch.enable_grad, torch.no_grad, torch.inference_mode):
            cache, table = K.new_cache(3, 2, 16, 64), torch.zeros((1, 2), dtype=torch.int32, device="cuda")
            w = torch.ones((), device="cuda", requires_grad=True)
            y = (w * cache).sum()
            before = cache._version
            with mode():
                write(cache, table)
            assert cache._version > before
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                y.backward()
    assert table._version > 0
    with torch.inference_mode():                # made there: no versions, and none asked for
        cache = K.new_cache(3, 2, 16, 64)
        K.move_pages(cache, torch.tensor([[0, 1]], dtype=torch.int32))
        assert not cache.any()
