"""Weights of logits that are large for their temperature: exp((x - max) / t) in 64 bits, where x / t and max / t have lost
what lies between them."""
import numpy as np
import pytest

from tests.test_gpu_sample import check
from vllm_sly_radiance_amd import _native_decode as N

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return N.lib()


def borders(rng, top, gap, n):
    """n temperatures, and min-p numbers in fp32 that lie next to the weight of top - gap, within 2^-28 of it and not
    within 2^-40: (temperatures, numbers); the weight is at least the number in some and not in others."""
    t = rng.uniform(gap * 0.05, gap * 0.08, 40000).astype(np.float32)
    w = np.exp(-gap / t.astype(np.float64))
    mp = w.astype(np.float32)
    off = np.abs(w - mp.astype(np.float64)) / w
    fine = (off < 2.0 ** -28) & (off > 2.0 ** -40)
    assert fine.sum() >= n
    return t[fine][:n], mp[fine][:n]


# (largest logit, the distance of the next): the ends of fp32's whole numbers, and both signs
@pytest.mark.parametrize("top,gap", [(2.0 ** 24 - 1, 1.0), (-(2.0 ** 23) - 1, 1.0), (1e6, 0.5), (3e30, 2.0 ** 78)])
@pytest.mark.parametrize("V", [60, 40000])
def test_weights_next_to_min_p(top, gap, V):
    rng = np.random.default_rng(int(V + abs(top) % 1000))
    rows = 60
    top = float(np.float32(top))
    assert float(np.float32(top - gap)) == top - gap
    t, mp = borders(rng, top, gap, rows)
    x = np.full((rows, V), -np.inf, np.float32)
    x[:, 7], x[:, V - 9] = top, top - gap
    assert V < 1000 or N.sample_workspace(rows, V, 0, 0) > 0        # (in parts)
    # the last element of any weight: the second where min-p leaves it
    for kw in (dict(), dict(p=[0.9999999] * rows)):
        tokens = check(x, np.ones(rows), t=t, mp=mp, **kw).cpu().numpy()
        if not kw:
            assert 10 < (tokens == 7).sum() < 50


def test_ordinary_logits_stay_as_they_are():
    rng = np.random.default_rng(3)
    x = (2.5 * rng.standard_normal((6, 3000))).astype(np.float32)
    check(x, rng.random(6), t=[0.3, 0.5, 0.7, 1.0, 1.3, 2.0], p=[0.9] * 6)
    check(x + np.float32(1000), rng.random(6), t=[0.3, 0.5, 0.7, 1.0, 1.3, 2.0], p=[0.9] * 6)
