"""Sampling on the GPU: the tokens that the definition in 64 bits picks."""
import numpy as np
import pytest
import torch

from oracle import decode_oracle as DO
from oracle import mxfp4_oracle as O
from tests._check import bf16_dev, to_dev
from vllm_sly_radiance_amd import _native_decode
from vllm_sly_radiance_amd import radiance_sample as S

pytestmark = pytest.mark.gpu

INF = np.inf
# Exponentials in fp32: of z = (x - top) log2 e, rounded twice, so off by 2^-23 |z| at most, which times ln 2 is the
# relative error of 2^z; with |z| 2^z below 1 (at |z| = 1.44 it is 0.53) the sum of n of them, which is at least
# 1, is off by less than sum 0.37 |z| 2^z 2^-22 / sum 2^z. Terms of |z| > 8 that dominate the sum are many and their
# errors' signs independent; bounded without that: |z| is at most log2 n where they matter (17 for 131072), so 17 ln 2
# 2^-23 < 2^-19. The instruction's own error, 2^-23, and sums of 32 terms in fp32, 2^-20 at the most, are below that
# again: 2^-18 in all.
LOGPROB = 2.0 ** -18


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_decode.lib()


def dev(x, dtype):
    return None if x is None else to_dev(np.asarray(x, dtype))


def check(x, u, t=None, k=None, p=None, mp=None, bf16=False):
    """x fp32 [rows, V] (bits of bf16 where that is asked for); parameters arrays of the rows or None."""
    x = np.asarray(x)
    values = O.bf16_to_f32(x) if bf16 else x.astype(np.float32)
    f = np.float32
    kw = dict(temperature=1.0 if t is None else dev(t, f), top_k=dev(k, np.int32), top_p=dev(p, f), min_p=dev(mp, f))
    logits = bf16_dev(x) if bf16 else to_dev(values)
    tokens = S.sample(logits, dev(u, f), **kw)
    again, lp = S.sample(logits, dev(u, f), logprobs=True, **kw)
    assert tokens.dtype == torch.int64 and torch.equal(tokens, again)
    at = lambda a, i, d: d if a is None else a[i]  # noqa: E731
    for i, row in enumerate(values):
        want, want_lp = DO.sample(row, float(f(u[i])), float(f(at(t, i, 1.0))), int(at(k, i, 0)),
                                  float(f(at(p, i, 1.0))), float(f(at(mp, i, 0.0))))
        assert int(tokens[i]) == want, f"row {i}"
        got = float(lp[i])
        assert np.isnan(got) if np.isnan(want_lp) else \
            got == want_lp or abs(got - want_lp) <= 2.0 ** -24 * abs(want_lp) + LOGPROB, f"row {i}"
    return tokens


def logits(rng, rows, V, spread=2.5):
    return (spread * rng.standard_normal((rows, V))).astype(np.float32)


SIZES = [1, 2, 7, 64, 1000, 4095, 4096, 4097, 50257, 131072]


@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("bf16", [False, True])
def test_every_filter(V, bf16):
    rng = np.random.default_rng(V + bf16)
    rows = 12
    x = logits(rng, rows, V)
    if bf16:
        x = O.f32_to_bf16(x)
    u = rng.random(rows)
    t, k = rng.uniform(0.3, 1.5, rows), rng.integers(0, min(V + 5, 400), rows)
    p, mp = rng.uniform(0.2, 1.1, rows), rng.uniform(-0.05, 0.2, rows)
    t[3] = 0
    for kw in (dict(), dict(t=t), dict(k=k), dict(p=p), dict(mp=mp), dict(t=t, k=k, p=p), dict(k=k, mp=mp),
               dict(t=t, k=k, p=p, mp=mp)):
        check(x, u, bf16=bf16, **kw)


@pytest.mark.parametrize("rows", [1, 3, 40, 300])
def test_rows(rows):
    rng = np.random.default_rng(rows)
    V = 3000
    check(logits(rng, rows, V), rng.random(rows), t=rng.uniform(0.5, 1, rows), k=rng.integers(1, 100, rows),
          p=rng.uniform(0.5, 1, rows))


def test_ties_go_to_the_lowest_index():
    rng = np.random.default_rng(1)
    x = np.zeros((8, 5000), np.float32)
    u = np.array([0, 0.25, 0.5, 0.999, 0.1, 0.3, 0.7, 0.9])
    check(x, u)                                             # all alike
    check(x, u, k=[1, 2, 3, 4096, 4097, 4999, 5000, 5001])
    assert check(x, u, k=[4] * 8).tolist() == [0, 1, 2, 3, 0, 1, 2, 3]
    check(x, u, p=[0.5, 0.25, 1e-9, 0.9999, 0.125, 0.0, -1.0, 1.0])
    check(x, u, mp=[1.0] * 8)
    assert check(x, u, t=[0] * 8).tolist() == [0] * 8
    few = rng.integers(-2, 3, (8, 20000)).astype(np.float32)        # thousands of ties at every value
    for k in (1, 17, 3000, 9000, 16001):
        check(few, u, k=[k] * 8, p=rng.uniform(0.3, 1, 8), t=rng.uniform(0.5, 2, 8))
    few[:, ::2] *= -1.0                                     # and zeros of both signs
    check(few, u, k=[9000] * 8)


def test_masked_rows():
    rng = np.random.default_rng(2)
    x = logits(rng, 9, 3001)
    x[1:] = np.where(rng.random((8, 3001)) < 0.99, -INF, x[1:])
    x[2] = -INF
    x[3] = -INF
    x[3, 2999] = -3e38
    x[4, :] = np.finfo(np.float32).min                      # the lowest finite value everywhere
    x[5, 17] = np.nan
    x[6, 100] = x[6, 2000] = INF
    x[7, :] = -INF
    x[7, [5, 6]] = INF
    u = rng.random(9)
    for kw in (dict(), dict(k=[5] * 9), dict(p=[0.7] * 9), dict(mp=[0.1] * 9), dict(k=[2900] * 9, p=[0.99] * 9),
               dict(t=[0] * 9), dict(t=[0.01] * 9), dict(t=[1e30] * 9, k=[50] * 9)):
        tokens = check(x, u, **kw)
        assert tokens[2] == -1 and tokens[5] == -1 and tokens[3] == 2999
    y = O.f32_to_bf16(x)
    check(y, u, k=[5] * 9, p=[0.7] * 9, bf16=True)


@pytest.mark.parametrize("t", [1e-30, 1e-3, 1e3, 1e30, INF, -1.0, -INF, np.nan])
def test_temperatures(t):
    rng = np.random.default_rng(3)
    x = logits(rng, 4, 2000)
    x[3, :1990] = -INF
    check(x, rng.random(4), t=[t] * 4)
    check(x, rng.random(4), t=[t] * 4, k=[3] * 4, p=[0.6] * 4, mp=[0.01] * 4)


def test_parameters_out_of_their_range():
    rng = np.random.default_rng(4)
    x, u = logits(rng, 6, 500), rng.random(6)
    check(x, u, k=[0, -1, 500, 501, 2 ** 31 - 1, -2 ** 31])
    check(x, u, p=[0, -3, 1, 2, np.nan, INF])
    check(x, u, mp=[0, -1, 1, 1.5, np.nan, INF])
    check(x, u, p=[1e-30, 1 - 2.0 ** -24, 0.5, 0.5, 0.5, 0.5], mp=[1e-30, 1e-30, 1e-38, 0.5, 1, 2])


def test_uniform_numbers():
    rng = np.random.default_rng(5)
    x = logits(rng, 8, 5000, spread=0.1)
    x[:, :3], x[:, -2:] = -INF, -INF
    u = [0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, np.nan, INF, 2.0 ** -60]
    tokens = check(x, u)
    assert tokens.tolist() == [3, 4997, 4997, 4997, 3, 3, 4997, 3]
    check(x, u, k=[100] * 8)


def test_numbers_for_all_rows():
    rng = np.random.default_rng(6)
    x, u = to_dev(logits(rng, 5, 900)), to_dev(rng.random(5).astype(np.float32))
    full = lambda v, d: torch.full((5,), v, dtype=d, device="cuda")  # noqa: E731
    a = S.sample(x, u, temperature=0.7, top_k=40, top_p=0.9, min_p=0.03)
    b = S.sample(x, u, temperature=full(0.7, torch.float32), top_k=full(40, torch.int32),
                 top_p=full(0.9, torch.float32), min_p=full(0.03, torch.float32))
    assert torch.equal(a, b)
    assert torch.equal(S.sample(x, u, temperature=0), x.argmax(1))
    assert torch.equal(S.sample(x, u), S.sample(x, u, temperature=1, top_k=0, top_p=1.0, min_p=0.0))


def test_strides():
    rng = np.random.default_rng(7)
    x, u = to_dev(logits(rng, 5, 901)), to_dev(rng.random(5).astype(np.float32))
    want = S.sample(x, u, top_k=30, top_p=0.9)
    for off in (0, 1, 2, 3):
        for dtype in (torch.float32, torch.bfloat16):
            wide = torch.full((5, 1023), 50.0, dtype=dtype, device="cuda")
            wide[:, off:off + 901] = x
            y = wide[:, off:off + 901]
            assert torch.equal(S.sample(y, u, top_k=30, top_p=0.9),
                               S.sample(y.contiguous(), u, top_k=30, top_p=0.9))
            if dtype == torch.float32:
                assert torch.equal(S.sample(y, u, top_k=30, top_p=0.9), want)
    assert torch.equal(S.sample(x.T.contiguous().T, u, top_k=30, top_p=0.9), want)
    assert torch.equal(S.sample(x[:1].expand(5, 901), u, top_k=30), S.sample(x[:1].repeat(5, 1), u, top_k=30))


def test_frequencies():
    """How often each token comes, over evenly spread uniform numbers, is its probability to within one."""
    n, p = 4096, np.array([0.5, 0.25, 0.125, 0.0625, 0.0625])
    x = np.full((1, 700), -INF, np.float32)
    where = [3, 650, 5, 400, 699]
    x[0, where] = np.log(p)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    tokens = S.sample(to_dev(np.repeat(x, n, 0)), to_dev(u)).cpu().numpy()
    for w, q in zip(where, p):
        assert abs((tokens == w).sum() - n * q) <= 1


def test_captured_and_on_streams():
    rng = np.random.default_rng(8)
    mk = lambda: (to_dev(logits(rng, 6, 20000)), to_dev(rng.random(6).astype(np.float32)))  # noqa: E731
    kw = dict(top_k=torch.full((6,), 900, dtype=torch.int32, device="cuda"), top_p=0.95, min_p=0.001, logprobs=True)
    (x, u), (x2, u2) = mk(), mk()
    S.sample(x, u, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = S.sample(x, u, **kw)
        out2 = S.sample(x2, u2, **kw)
    side = torch.cuda.Stream()
    for _ in range(4):
        for dst, src in zip((x, u, x2, u2), mk() + mk()):
            dst.copy_(src)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = S.sample(x, u, **kw)
        want2 = S.sample(x2, u2, **kw)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out + out2, want + want2):
            assert torch.equal(a, b)


def test_no_rows():
    e = torch.empty((0, 50), device="cuda")
    assert S.sample(e, torch.empty(0, device="cuda")).shape == (0,)
    t, lp = S.sample(e, torch.empty(0, device="cuda"), logprobs=True)
    assert t.shape == lp.shape == (0,)


REFUSED = [
    (dict(logits=lambda x, u: x.half()), "logits must be fp32 or bf16"), (dict(logits=lambda x, u: x[0]), "logits must"),
    (dict(logits=lambda x, u: x[:, :0]), "no vocabulary"), (dict(uniform=lambda x, u: u[:2]), "uniform must be fp32 .3."),
    (dict(uniform=lambda x, u: u.double()), "uniform must be fp32"),
    (dict(temperature=lambda x, u: u[:1]), "temperature must be fp32"),
    (dict(top_k=lambda x, u: u), "top_k must be int32"), (dict(top_p=lambda x, u: u.long()), "top_p must be fp32"),
    (dict(min_p=lambda x, u: u.cpu()), "cuda:0 and cpu"), (dict(top_k=lambda x, u: 1 << 40), "top_k"),
]


@pytest.mark.parametrize("change,words", REFUSED, ids=lambda x: "-".join(x) if isinstance(x, dict) else "")
def test_refused(change, words):
    x, u = torch.randn((3, 50), device="cuda"), torch.rand(3, device="cuda")
    kw = dict(logits=x, uniform=u)
    kw.update({n: f(x, u) for n, f in change.items()})
    with pytest.raises(RuntimeError, match=words):
        S.sample(**kw)
    assert torch.equal(S.sample(x, u, temperature=0), x.argmax(1))
