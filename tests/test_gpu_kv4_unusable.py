"""Attention over the 4-bit cache where pages cannot be read: caches of no pages, page numbers outside the
cache. What a query does not see has no effect on it."""
import numpy as np
import pytest
import torch

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
