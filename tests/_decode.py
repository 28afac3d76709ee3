"""Shared helpers of the tests of the convolution, the delta rule and sampling."""
import numpy as np
import torch

from oracle import decode_oracle as DO
from oracle import mxfp4_oracle as O
from tests._check import bf16_dev, to_dev


def bits(rng, *shape, scale=1.0):
    return O.f32_to_bf16((scale * rng.standard_normal(shape)).astype(np.float32))


def f64(b):
    """bf16 bits as float64."""
    return O.bf16_to_f32(b).astype(np.float64)


def host(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def i32(a):
    return to_dev(np.asarray(a, np.int32))


def starts_of(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


class Delta:
    """A batch for the delta rule: arrays as the device gets them, and the definition."""

    def __init__(self, rng, lens, heads, slots=None, read=None, extra_rows=0, v_scale=1.0, a_scale=1.0):
        Hk, Hv, dk, dv = heads
        self.lens, self.heads = list(lens), heads
        T = sum(lens) + extra_rows
        self.q, self.k = bits(rng, T, Hk, dk), bits(rng, T, Hk, dk)
        self.v = bits(rng, T, Hv, dv, scale=v_scale)
        self.a, self.b = bits(rng, T, Hv, scale=a_scale), bits(rng, T, Hv)
        self.a_log = np.log(rng.uniform(0.5, 16, Hv)).astype(np.float32)
        step = np.exp(rng.uniform(np.log(1e-3), np.log(0.1), Hv))
        self.dt_bias = (step + np.log(-np.expm1(-step))).astype(np.float32)
        B = len(lens)
        self.slots = slots or B + 2
        self.state = (0.3 * rng.standard_normal((self.slots, Hv, dk, dv))).astype(np.float32)
        self.write = rng.permutation(self.slots)[:B].astype(np.int32)
        self.read = self.write.copy() if read is None else np.asarray(read, np.int32)

    def expect(self, **kw):
        n = sum(self.lens)
        return DO.delta(f64(self.q)[:n], f64(self.k)[:n], f64(self.v)[:n], f64(self.a)[:n], f64(self.b)[:n],
                        self.a_log.astype(np.float64), self.dt_bias.astype(np.float64),
                        self.state.astype(np.float64), self.lens, self.read, **kw)

    def device(self, write=None, max_q=None):
        """Arguments of gated_delta_rule; the state is the eighth."""
        return [bf16_dev(self.q), bf16_dev(self.k), bf16_dev(self.v), bf16_dev(self.a), bf16_dev(self.b),
                to_dev(self.a_log), to_dev(self.dt_bias), to_dev(self.state), i32(starts_of(self.lens)),
                i32(self.read), i32(self.write if write is None else write),
                max(self.lens, default=0) if max_q is None else max_q]

    def check(self, out, state, write=None, **kw):
        """Outputs and all slots against the definition; returns the worst errors over their bounds."""
        ref, tol, states, bounds = self.expect(**kw)
        n = sum(self.lens)
        worst = float((np.abs(host(out)[:n] - ref) / tol).max()) if n else 0.0
        assert worst <= 1, f"outputs are {worst:.3g} times their bound off"
        got, want = host(state), self.state.astype(np.float64)
        write = self.write if write is None else write
        touched = {}
        for b, m in enumerate(self.lens):
            if write.ndim == 1:
                touched[int(write[b])] = (states[b][m], bounds[b][m])
            else:
                for i in range(min(m, write.shape[1])):
                    touched[int(write[b, i])] = (states[b][i + 1], bounds[b][i + 1])
        worst_state = 0.0
        for s in range(self.slots):
            if s in touched:
                S, E = touched[s]
                off = np.sqrt(((got[s] - S) ** 2).sum(1))
                worst_state = max(worst_state, float((off / (E + 2.0 ** -100)).max()))
            else:
                assert np.array_equal(got[s], want[s]), f"slot {s} was written"
        assert worst_state <= 1, f"states are {worst_state:.3g} times their bound off"
        return worst, worst_state


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))
