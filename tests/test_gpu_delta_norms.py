"""Keys and queries of every length that bf16 holds: the delta rule divides by it, in whichever form."""
import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as O
from tests._decode import Delta, host
from vllm_sly_radiance_amd import _native_decode
from vllm_sly_radiance_amd import radiance_gdn as G

pytestmark = pytest.mark.gpu

STEPS, CHUNKS = 1, 4096         # max_q: token after token, in chunks


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_decode.lib()


def scaled(d, what, scale, rows=slice(None)):
    x = getattr(d, what)
    x[rows] = O.f32_to_bf16((O.bf16_to_f32(x[rows]).astype(np.float64) * scale).astype(np.float32))


@pytest.mark.parametrize("scale", [1e36, 1e25, 1e16, 1e-16, 1e-25, 1e-36], ids=str)
@pytest.mark.parametrize("what", ["q", "k", "qk"])
@pytest.mark.parametrize("eps", [1e-6, 0.0], ids=str)
def test_lengths_token_after_token(scale, what, eps):
    """Rows whose squares leave the range of fp32 have the direction that they have."""
    d = Delta(np.random.default_rng(41), [9, 3], (2, 4, 128, 128))
    for w in what:
        scaled(d, w, scale)
    args = d.device(max_q=STEPS)
    d.check(G.gated_delta_rule(*args, eps=eps), args[7], eps=eps)


def test_long_keys_meet_large_states():
    """A key's product with the state, 1e16 times 1e30, is divided by the key's length."""
    for max_q in (STEPS, CHUNKS):
        d = Delta(np.random.default_rng(42), [70], (1, 2, 128, 128), v_scale=1e30)
        scaled(d, "k", 1e16)
        d.state *= np.float32(1e30)
        args = d.device(max_q=max_q)
        d.check(G.gated_delta_rule(*args), args[7])
