"""The convolution, the delta rule, the gated norm, attention and sampling together, through the example: however
a sequence's tokens reach its states (one chunk, several, one by one, through a fork, beside others, drafted
and in part rejected), the logits of its last token agree."""
import numpy as np
import pytest
import torch

from examples.gdn_generate import Hybrid, main
from vllm_sly_radiance_amd import _native, _native_decode, _native_kv4

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native.lib(), _native_kv4.lib(), _native_decode.lib()


def close(a, b):
    # Pieces of different lengths go through other kernels, whose fp32 results differ by some 1e-5 and whose bf16
    # outputs then may take the neighbour. In e4m3, per token, that is at most a step of 2^-3 of an element, in
    # the one element of 2^-8 / 1e-5 = 400 or fewer of them that lies so near a boundary: 2^-3 / 20 = 0.6 % of a
    # product's norm a quantization, of which this stack has two a layer. A key or value near the middle
    # of two codes in 4 bits takes the other: at most 1/3 of a channel's block maximum, in one token of many.
    rel = float((a - b).norm() / b.norm())
    assert rel < 0.05, rel


@torch.no_grad()
def test_ways_into_the_states_agree():
    s = Hybrid(layers=4, pages=96)
    rng = np.random.default_rng(3)
    tokens = rng.integers(0, 512, 330).tolist()
    other = rng.integers(0, 512, 41).tolist()
    a = s.add()
    want = s.forward([a], [tokens])[-1]
    s.drop(a)

    b, c = s.add(), s.add()
    s.forward([b], [tokens[:200]])
    s.forward([c, b], [other, tokens[200:323]])
    d = s.fork(b)
    s.forward([b, d], [tokens[323:324], other[:5]])      # d goes its own way
    # drafted tokens: all rejected, then one of three right, then all of them
    s.forward([d, b], [other[5:8], tokens[324:325] + other[:2]], drafts=True)
    s.keep(d, 2, 1)
    s.keep(b, 2, 0)
    s.forward([b], [tokens[325:327] + other[:2]], drafts=True)
    s.keep(b, 3, 1)
    s.forward([b], [tokens[327:329]], drafts=True)
    s.keep(b, 1, 1)
    e = s.fork(b)
    got = s.forward([b, d, e], [tokens[329:], other[8:9], tokens[329:]])
    close(got[0], want)
    close(got[2], want)
    assert float((got[1] - want).norm() / want.norm()) > 0.5


def test_example_runs():
    s, ids, prompt, out = main(["--layers", "4", "--prompt", "150", "--steps", "9"])
    for sequence, o in zip(ids, out):
        assert s.pool.length(sequence) == len(prompt) + len(o) and len(o) >= 9
        assert all(0 <= t < 512 for t in o)
