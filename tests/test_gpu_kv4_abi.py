"""The C ABI of the 4-bit cache on device addresses of the least alignment that it asks for: 16 bytes, none of
them a multiple of 32."""
import numpy as np
import pytest
import torch

from tests._check import stream
from tests._kv4 import Batch
from vllm_sly_radiance_amd import _native_kv4 as N

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return N.lib()


def odd(t):
    """A copy whose first byte is 16 past a multiple of 32, and its address."""
    raw = torch.zeros(t.numel() * t.element_size() + 64, dtype=torch.uint8, device="cuda")
    at = 16 if raw.data_ptr() % 32 == 0 else 0
    x = raw[at:at + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
    x.copy_(t)
    assert x.data_ptr() % 32 == 16
    return x


@pytest.mark.parametrize("d,lens,qs", [(256, [3000, 40, 2100], [1, 1, 2]), (128, [3000, 40], [1, 4]),
                                       (64, [2900, 77], [1, 3]), (256, [300, 280], [250, 270])])
def test_attention(d, lens, qs):
    b = Batch(np.random.default_rng(d), lens, qs, 32, 4, d, 16)
    q, cache, table, dl, starts, mq, ml = b.device()
    q, cache = odd(q), odd(cache)
    out = odd(torch.full_like(q, 7.0))
    need = N.attention_workspace(len(q), len(lens), mq, ml, 32, 4, d, 0)
    space = odd(torch.zeros(need // 4 + 4, dtype=torch.float32, device="cuda"))
    print(f"[kv4] odd addresses d={d} lens={lens}", flush=True)
    N.check(N.lib().kv4_attention(
        q.data_ptr(), q.stride(0), q.stride(1), cache.data_ptr(), cache.shape[0], cache.stride(0), 16,
        table.data_ptr(), table.stride(0), table.shape[1], dl.data_ptr(), starts.data_ptr(), out.data_ptr(),
        space.data_ptr(), need, len(q), len(lens), mq, ml, 32, 4, d, d ** -0.5, 0, N.CAUSAL, stream()))
    torch.cuda.synchronize()
    b.check(out)
