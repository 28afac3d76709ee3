"""PagePool.extend is all or nothing also where the copy of a shared page or the step's buffers fail."""
import numpy as np
import pytest
import torch

from vllm_sly_radiance_amd import kv4_pool
from vllm_sly_radiance_amd import radiance_kv4 as K
from vllm_sly_radiance_amd.kv4_pool import PagePool


def state(pool):
    return ([(i, pool.pages_of(i), pool.length(i)) for i in pool._sequences], pool.free_pages, sorted(pool._free),
            list(pool._refs))


@pytest.mark.parametrize("what", ["move", "step"])
def test_extend_that_fails_changes_nothing(monkeypatch, what):
    pool = PagePool(K.new_cache(12, 1, 16, 64, device="cpu", layers=2))
    moved = []
    monkeypatch.setattr(kv4_pool._kv4, "move_pages", lambda cache, pairs, table=None: moved.extend(pairs.tolist()))
    a, b = pool.add(), pool.add()
    pool.extend([a, b], [20, 16])
    c, d = pool.fork(a), pool.fork(a)
    before = state(pool)

    def fail(*args, **kwargs):
        raise RuntimeError("out of memory")
    with monkeypatch.context() as m:
        if what == "move":
            m.setattr(kv4_pool._kv4, "move_pages", fail)
        else:
            m.setattr(kv4_pool.torch, "empty", fail)
        with pytest.raises(RuntimeError, match="out of memory"):
            pool.extend([a, b, c, d], [30, 5, 1, 0])
    assert state(pool) == before
    step = pool.extend([a, b, c, d], [30, 5, 1, 0])
    assert step.seq_lens.tolist() == [50, 21, 21, 20] and len(moved) >= 1
    assert len(set(step.slots.tolist())) == 36 and torch.equal(step.q_starts, torch.tensor([0, 30, 35, 36, 36],
                                                                                          dtype=torch.int32))
    used = np.concatenate([pool.pages_of(i) for i in (a, b, c, d)])
    assert pool.free_pages == 12 - len(set(used.tolist()))
