"""Sampling of few rows of a large vocabulary, which several workgroups share: the tokens that the definition in 64
bits picks, whatever part of the row holds what, and those that one workgroup a row picks."""
import numpy as np
import pytest
import torch

from oracle import decode_oracle as DO
from oracle import mxfp4_oracle as O
from tests._check import bf16_dev, to_dev
from tests.test_gpu_sample import LOGPROB
from vllm_sly_radiance_amd import _native_decode as N
from vllm_sly_radiance_amd import radiance_sample as S

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return N.lib()


# Weights are added as whole numbers of 2^-s, s = 62 - ceil(log2 V) (45 for 131072): each is off by half of one at most,
# a sum of V of them by V 2^-(s + 1). The largest weight is 1, so that uniform times the sum, and the sum up to an
# element, are those of a uniform number no further away than 2 V 2^-(s + 1). The token's index grows with it.
def pick(row, u, *how):
    off = len(row) * 2.0 ** -(62 - int(np.ceil(np.log2(len(row)))))
    return DO.sample(row, max(u - off, 0.0), *how)[0], DO.sample(row, u + off, *how)[0]


def log_prob(row, token):
    row = row.astype(np.float64)
    with np.errstate(invalid="ignore"):
        z = np.where(row == row.max(), 0.0, row - row.max())
    return z[token] - np.log(np.exp(z).sum())


def check(x, u, bf16=False, **kw):
    values = O.bf16_to_f32(x) if bf16 else x
    logits = bf16_dev(x) if bf16 else to_dev(x)
    f = lambda v: v if isinstance(v, (int, float)) else to_dev(np.asarray(v, np.float32))  # noqa: E731
    args = {n: f(v) for n, v in kw.items()}
    tokens, lp = S.sample(logits, to_dev(np.asarray(u, np.float32)), logprobs=True, **args)
    assert torch.equal(tokens, S.sample(logits, to_dev(np.asarray(u, np.float32)), **args))
    of = lambda n, i, d: d if n not in kw else float(np.float32(  # noqa: E731
        kw[n] if isinstance(kw[n], (int, float)) else kw[n][i]))
    for i, row in enumerate(values):
        how = of("temperature", i, 1.0), int(of("top_k", i, 0)), of("top_p", i, 1.0), of("min_p", i, 0.0)
        want, want_lp = DO.sample(row, float(np.float32(u[i])), *how)
        got, token = float(lp[i]), int(tokens[i])
        if token != want:
            low, high = pick(row, float(np.float32(u[i])), *how)
            assert 0 <= low <= token <= high, f"row {i}: {token}, not {want}"
            want_lp = log_prob(row, token)
        assert np.isnan(got) if np.isnan(want_lp) else \
            got == want_lp or abs(got - want_lp) <= 2.0 ** -24 * abs(want_lp) + LOGPROB, f"row {i}"
    return tokens


def in_parts(rows, V, bf16, top_k=0):
    return N.sample_workspace(rows, V, top_k, N.BF16 if bf16 else 0) > 0


# (rows, vocabulary, bf16): two parts of the smallest rows that have any, a last part that is short, eight parts, and
# rows that begin at every alignment
@pytest.mark.parametrize("rows,V,bf16", [(1, 32768, False), (1, 65536, True), (5, 50257, False), (3, 131071, True),
                                         (9, 131073, False), (128, 33000, False), (2, 400001, False)])
def test_filters(rows, V, bf16):
    assert in_parts(rows, V, bf16) and not in_parts(rows, V, bf16, 512)
    rng = np.random.default_rng(V)
    x = (2.5 * rng.standard_normal((rows, V))).astype(np.float32)
    if bf16:
        x = O.f32_to_bf16(x)
    u = rng.random(rows)
    few = rows <= 9
    for kw in (dict(top_p=0.9), dict(top_p=rng.uniform(0.3, 1.2, rows), temperature=rng.uniform(0.4, 1.4, rows)),
               dict(), dict(min_p=0.01), dict(top_k=2000, temperature=0.8), dict(top_k=700, top_p=0.8, min_p=0.02),
               dict(top_p=0.999999, min_p=0.001), dict(top_k=50, top_p=0.9))[:None if few else 2]:
        check(x, u, bf16=bf16, **kw)


def test_values_that_only_some_parts_have():
    V = 131072
    rng = np.random.default_rng(4)
    x = (2 * rng.standard_normal((10, V))).astype(np.float32)
    x[0, V - 1] = np.nan                            # the last part
    x[1] = -np.inf
    x[2, :V - 3] = -np.inf                          # parts of -infinity only
    x[3, 100:] = -np.inf
    x[4, [5, V // 2, V - 2]] = np.inf
    x[5] = 0.25                                     # one value: no steps, and every element a tie
    x[6] = np.round(x[6])                           # ties across parts, more of them than the list holds
    x[7, ::2] = -3e38
    x[8] = np.where(rng.random(V) < 0.999, -np.inf, x[8])
    x[9, 70000] = 60.0                              # one logit that has all the weight
    u = rng.random(10)
    t = np.full(10, 0.9)
    for kw in (dict(top_p=0.9), dict(), dict(top_k=1000, top_p=0.95), dict(top_k=600), dict(top_p=0.0), dict(top_p=1e-3, min_p=0.5),
               dict(temperature=t, top_p=0.7), dict(temperature=np.where(np.arange(10) % 3, 1.0, 0.0), top_p=0.7),
               dict(temperature=0.02, top_p=0.9), dict(temperature=300.0, top_p=0.5)):
        check(x, u, **kw)
        check(x, np.where(u < 0.5, 0.0, 1.0 - 2.0 ** -24), **kw)


def test_parts_and_whole_rows_agree():
    """A row among 4 others goes in parts, among 200 in one piece: the same token, and a log probability whose
    sum is taken in another order."""
    V = 40000
    rng = np.random.default_rng(6)
    x = to_dev((2 * rng.standard_normal((200, V))).astype(np.float32))
    u = to_dev(rng.random(200).astype(np.float32))
    assert in_parts(4, V, False) and not in_parts(200, V, False)
    for kw in (dict(top_p=0.92, temperature=0.7), dict(), dict(top_k=900)):
        whole, lp = S.sample(x, u, logprobs=True, **kw)
        for i in range(0, 200, 40):
            some, lp4 = S.sample(x[i:i + 4], u[i:i + 4], logprobs=True, **kw)
            assert torch.equal(some, whole[i:i + 4])
            assert torch.allclose(lp4, lp[i:i + 4], rtol=2.0 ** -23, atol=2 * LOGPROB)


def test_strided_rows_and_a_graph():
    V = 50000
    rng = np.random.default_rng(8)
    wide = to_dev((2 * rng.standard_normal((6, V + 5))).astype(np.float32))
    x = wide[:, 3:V + 3]                            # rows at odd addresses, V + 5 apart
    u = to_dev(rng.random(6).astype(np.float32))
    how = dict(top_p=0.9, min_p=0.001, temperature=0.8)
    want = S.sample(x.contiguous(), u, **how)
    assert torch.equal(S.sample(x, u, **how), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        S.sample(x, u, **how)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, lp = S.sample(x, u, logprobs=True, **how)
    for i in range(4):
        wide.copy_(to_dev((2 * rng.standard_normal((6, V + 5))).astype(np.float32)))
        u.copy_(to_dev(rng.random(6).astype(np.float32)))
        tokens, p = S.sample(x, u, logprobs=True, **how)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, tokens) and torch.equal(lp, p)
