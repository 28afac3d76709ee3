"""The short causal convolution on the GPU against its definition in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import decode_oracle as DO
from tests._check import bf16_dev, host_u16
from tests._decode import bits, f64, host, i32, same, starts_of
from vllm_sly_radiance_amd import _native_decode
from vllm_sly_radiance_amd import radiance_gdn as G

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_decode.lib()


class Conv:
    def __init__(self, rng, lens, C, W, bias=True, slots=None):
        self.lens, self.C, self.W = list(lens), C, W
        self.x, self.w = bits(rng, sum(lens), C), bits(rng, C, W)
        self.bias = bits(rng, C) if bias else None
        self.slots = slots or len(lens) + 2
        self.state = bits(rng, self.slots, W - 1, C)
        self.write = rng.permutation(self.slots)[:len(lens)].astype(np.int32)
        self.read = self.write.copy()

    def device(self, write=None, max_q=None):
        return [bf16_dev(self.x), bf16_dev(self.w), None if self.bias is None else bf16_dev(self.bias),
                bf16_dev(self.state), i32(starts_of(self.lens)), i32(self.read),
                i32(self.write if write is None else write),
                max(self.lens, default=0) if max_q is None else max_q]

    def check(self, out, state, write=None, silu=True):
        ref, tol, seen = DO.conv(f64(self.x), f64(self.w), None if self.bias is None else f64(self.bias),
                                 f64(self.state), self.lens, self.read, silu)
        got = host(out)
        fine = np.isfinite(ref)
        assert (np.isfinite(got) == fine).all() and (np.abs(got - ref)[fine] <= tol[fine]).all()
        want = f64(self.state)
        write = self.write if write is None else write
        for b, n in enumerate(self.lens):
            if write.ndim == 1:
                if 0 <= write[b] < self.slots:
                    want[write[b]] = seen[b][n:]
            else:
                for i in range(min(n, write.shape[1])):
                    want[write[b, i]] = seen[b][i + 1:i + self.W]
        assert np.array_equal(host(state), want, equal_nan=True)


@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("C", [8, 264, 4104])
@pytest.mark.parametrize("lens", [[1], [1] * 7, [2, 0, 3, 1], [15, 16, 17, 0, 33], [200, 1]], ids=str)
def test_against_the_definition(lens, C, W):
    c = Conv(np.random.default_rng(W + C + sum(lens)), lens, C, W, bias=W != 3)
    for max_q in (None, 1, 100):
        args = c.device(max_q=max_q)
        c.check(G.causal_conv(*args), args[3])


def test_without_silu():
    c = Conv(np.random.default_rng(1), [20, 3], 64, 4)
    args = c.device()
    c.check(G.causal_conv(*args, silu=False), args[3], silu=False)


@pytest.mark.parametrize("lens,cols", [([8, 8], 8), ([5, 1, 0, 2], 5), ([40, 3], 3)])
def test_the_state_after_each_token(lens, cols):
    c = Conv(np.random.default_rng(2), lens, 72, 4, slots=len(lens) * cols + 1)
    write = np.random.default_rng(3).permutation(c.slots)[:len(lens) * cols].reshape(len(lens), cols)
    c.read = write[:, -1].astype(np.int32)
    args = c.device(write)
    c.check(G.causal_conv(*args), args[3], write)


def test_slots():
    """New sequences, forks, states nobody wants, slots past the pool (NaN, where the state reaches)."""
    c = Conv(np.random.default_rng(4), [20, 2, 0, 30, 1], 64, 4, slots=7)
    c.read = np.array([-1, 5, 5, 9, 2], np.int32)
    write = np.array([3, 6, 0, 8, -1], np.int32)
    args = c.device(write)
    c.check(G.causal_conv(*args), args[3], write)


def test_views():
    c = Conv(np.random.default_rng(5), [20, 3], 64, 4)
    args = c.device()
    want = G.causal_conv(*args)
    T = 23
    wide = torch.zeros((T, 104), dtype=torch.bfloat16, device="cuda")
    states = torch.zeros((c.slots, 2, 3, 64), dtype=torch.bfloat16, device="cuda")
    for place in (8, 20):                       # aligned, and copied first
        new = c.device()
        wide[:, place:place + 64] = new[0]
        states[:, 1] = new[3]
        new[0], new[3] = wide[:, place:place + 64], states[:, 1]
        assert torch.equal(G.causal_conv(*new), want)
        assert torch.equal(states[:, 1], args[3]) and not states[:, 0].any()
    new = c.device()
    new[1] = new[1].T.contiguous().T
    assert torch.equal(G.causal_conv(*new), want)


def test_not_finite_inputs_reach_their_window():
    c = Conv(np.random.default_rng(6), [40], 16, 4)
    c.x[10, 3], c.x[20, 5] = 0x7FC0, 0x7F80
    args = c.device()
    out = host(G.causal_conv(*args))
    bad = ~np.isfinite(out)
    assert bad[10:14, 3].all() and bad[:, 3].sum() == 4
    # infinity: SiLU of -infinity is not a number, of infinity is infinity
    assert set(np.nonzero(bad[:, 5])[0]) == set(range(20, 24))
    assert bad.sum() == 8


def test_large_sums():
    """SiLU far out on both sides."""
    c = Conv(np.random.default_rng(7), [50], 64, 4)
    c.w = bits(np.random.default_rng(8), 64, 4, scale=60.0)
    args = c.device()
    c.check(G.causal_conv(*args), args[3])


def test_captured_and_on_streams():
    c = Conv(np.random.default_rng(9), [20, 1, 3], 64, 4)
    eager, held = c.device(), c.device()
    G.causal_conv(*c.device())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = G.causal_conv(*held)
    held[3].copy_(eager[3])
    side = torch.cuda.Stream()
    for i in range(4):
        src = Conv(np.random.default_rng(10 + i), [3, 20, 1] if i % 2 else [20, 1, 3], 64, 4).device()
        for j in (0, 1, 2, 4, 5, 6):
            eager[j].copy_(src[j]), held[j].copy_(src[j])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = G.causal_conv(*eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and same(held[3], eager[3])


def test_nothing_to_do_and_rows_of_no_sequence():
    c = Conv(np.random.default_rng(11), [], 16, 3)
    assert G.causal_conv(*c.device()).shape == (0, 16)
    c = Conv(np.random.default_rng(12), [4], 16, 3)
    args = c.device()
    args[4] = i32([1, 3])
    before = G.causal_conv(*c.device())
    del before
    out = G.causal_conv(*args)
    c.lens, c.x = [2], c.x[1:3]
    c.check(out[1:3], args[3])


REFUSED = [
    (0, lambda a: a[0].float(), "x must be bf16"), (0, lambda a: a[0][0], "x must be"),
    (0, lambda a: a[0][:, :12], "multiple of 8"), (1, lambda a: a[1][:, :1], "width 1|state must be"),
    (1, lambda a: a[1].float(), "weight must be bf16"), (2, lambda a: a[2][:8], "bias must be bf16"),
    (3, lambda a: a[3][:, :2], "state must be bf16"), (3, lambda a: a[3].float(), "state must be bf16"),
    (3, lambda a: a[3].transpose(1, 2).contiguous().transpose(1, 2), "contiguous"),
    (4, lambda a: a[4][:1], "q_starts"), (5, lambda a: a[5].long(), "read_slots"),
    (6, lambda a: a[6][:1], "write_slots"), (7, lambda a: -2, "max_q=-2"), (2, lambda a: a[2].cpu(), "cpu"),
]


@pytest.mark.parametrize("at,change,words", REFUSED)
def test_refused(at, change, words):
    c = Conv(np.random.default_rng(13), [2, 1], 16, 4)
    args = c.device()
    bad = list(args)
    bad[at] = change(args)
    with pytest.raises(RuntimeError, match=words):
        G.causal_conv(*bad)
    c.check(G.causal_conv(*args), args[3])
    assert host_u16(args[0]).shape == (3, 16)
