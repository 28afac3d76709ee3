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


@pytest.mark.parametrize("scale", [1e25, 1e-25], ids=str)
@pytest.mark.parametrize("what", ["q", "k", "qk"])
def test_lengths_beside_a_value_that_is_not_finite(scale, what):
    """A chunk with NaN in it goes token after token: the channels and the tokens that the NaN does not reach are
    what they are without it."""
    d = Delta(np.random.default_rng(43), [100], (1, 2, 128, 128))
    for w in what:
        scaled(d, w, scale)
    for eps in (1e-6, 0.0):
        ref, tol, states, bounds = d.expect(eps=eps)
        args = d.device(max_q=CHUNKS)
        args[2][70, 1, 7] = float("nan")
        out, state = host(G.gated_delta_rule(*args, eps=eps)), host(args[7])[d.write[0]]
        hit = np.zeros(out.shape, bool)
        hit[70:, 1, 7] = True
        assert np.isnan(out[hit]).all() and (np.abs(out - ref)[~hit] <= tol[~hit]).all()
        off = np.sqrt(((state - states[0][-1]) ** 2).sum(1))
        bad = np.zeros(off.shape, bool)
        bad[1, 7] = True
        assert np.isnan(off[bad]).all() and (off[~bad] <= bounds[0][-1][~bad]).all()


# A row of length s far below sqrt(eps) counts as one of length s / sqrt(eps), in which outputs (of queries) and states (from
# zeros, of keys) are linear: their bounds are those for length 1 times that.
def unit_length(x, eps):
    return np.minimum(np.sqrt((O.bf16_to_f32(x).astype(np.float64) ** 2).sum(-1) / eps), 1.0)


@pytest.mark.parametrize("max_q", [STEPS, CHUNKS])
@pytest.mark.parametrize("scale", [1e-6, 1e-16, 1e-20, 1e-25, 1e-30], ids=str)
@pytest.mark.parametrize("eps", [1e-6, 1e-2], ids=str)
def test_short_queries_beside_eps(scale, eps, max_q):
    """(Of a state that no token adds to: beta is 0.)"""
    d = Delta(np.random.default_rng(44), [70], (1, 2, 128, 128))
    scaled(d, "q", scale)
    d.b[:] = 0xFF80                                 # -infinity
    args = d.device(max_q=max_q)
    out = host(G.gated_delta_rule(*args, eps=eps))
    ref, tol, *_ = d.expect(eps=eps)
    half = 2.0 ** -8 * np.abs(ref)
    assert (np.abs(out - ref) <= (tol - half) * unit_length(d.q, eps)[..., None] + half + 2.0 ** -126).all()


@pytest.mark.parametrize("max_q", [STEPS, CHUNKS])
@pytest.mark.parametrize("scale", [1e-6, 1e-16, 1e-20, 1e-25, 1e-30], ids=str)
def test_short_keys_beside_eps(scale, max_q):
    d = Delta(np.random.default_rng(45), [70], (1, 2, 128, 128), read=[-1])
    scaled(d, "k", scale)
    args = d.device(max_q=max_q)
    G.gated_delta_rule(*args)
    *_, states, bounds = d.expect()
    off = np.sqrt(((host(args[7])[d.write[0]] - states[0][-1]) ** 2).sum(1))
    assert (off <= bounds[0][-1] * unit_length(d.k, 1e-6).max() + 2.0 ** -126).all()


@pytest.mark.parametrize("scale", [1e36, 1e25, 1e16, 1e-16, 1e-25, 1e-36], ids=str)
@pytest.mark.parametrize("what", ["q", "k", "qk"])
@pytest.mark.parametrize("eps", [1e-6, 0.0], ids=str)
def test_lengths_in_chunks(scale, what, eps):
    d = Delta(np.random.default_rng(46), [90, 3], (2, 4, 128, 64))
    for w in what:
        scaled(d, w, scale)
    args = d.device(max_q=CHUNKS)
    d.check(G.gated_delta_rule(*args, eps=eps), args[7], eps=eps)
