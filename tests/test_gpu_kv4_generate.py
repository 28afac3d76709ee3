"""The operators of the 4-bit cache together, through the example: however a sequence's tokens reach the
cache (one chunk, several, one by one, through a fork, beside others, before and after a compaction), the
logits of its last token agree."""
import numpy as np
import pytest
import torch

from examples.kv4_generate import Stack, main
from vllm_sly_radiance_amd import _native, _native_kv4

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native.lib(), _native_kv4.lib()


def close(a, b):
    # Chunks of different length go through other kernels, whose bf16 outputs may differ in the last
    # place; a key or value near the middle of two codes then takes the other one. One such step is at
    # most half the largest code's spacing, 1/3 of a channel's block maximum, in one token of many.
    rel = float((a - b).norm() / b.norm())
    assert rel < 0.05, rel


@torch.no_grad()
def test_ways_into_the_cache_agree():
    s = Stack(layers=2, pages=96)
    rng = np.random.default_rng(3)
    tokens = rng.integers(0, 512, 330).tolist()
    other = rng.integers(0, 512, 41).tolist()
    a = s.pool.add()
    want = s.forward([a], [tokens])[-1]
    s.pool.free(a)

    b, c = s.pool.add(), s.pool.add()
    s.forward([b], [tokens[:200]])
    s.forward([c, b], [other, tokens[200:326]])
    d = s.pool.fork(b)
    s.forward([b, d], [tokens[326:327], other[:5]])     # d goes its own way on a copied page
    s.forward([b], [tokens[327:328]])
    s.pool.free(c)
    assert s.pool.compact() > 0
    s.forward([d, b], [other[5:6], tokens[328:329]])
    # drafted tokens that are rejected leave nothing behind
    n = s.pool.length(b)
    s.forward([b], [other[:9]])
    s.pool.truncate(b, n)
    e = s.pool.fork(b)
    got = s.forward([b, e], [tokens[329:], tokens[329:]])
    close(got[0], want)
    close(got[1], want)


def test_example_runs():
    s, ids, prompt, out = main(["--layers", "2", "--prompt", "150", "--steps", "9"])
    for sequence, o in zip(ids, out):
        assert s.pool.length(sequence) == len(prompt) + len(o) and len(o) >= 9
    assert out[0][0] != out[1][0]
