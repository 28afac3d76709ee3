"""Runs the convolution and the delta rule token after token, compiled for the CPU (tests/test_cpu_model.py), over batches
whose starts and slots hold anything. What they read and write ends, or begins, at memory that cannot be touched; where
starts are in order, the results are the definition's.

  python -m tests.cpu_model.sequences LIBRARY SEED
"""
import ctypes
import sys

import numpy as np

from oracle import decode_oracle as DO
from oracle import mxfp4_oracle as O
from tests.cpu_model.memory import Guarded, guarded

LOWEST, HIGHEST = -2 ** 31, 2 ** 31 - 1


def starts_of(rng, batch, total):
    kind = rng.integers(4)
    if kind == 0:
        return np.sort(rng.integers(0, total + 1, batch + 1))
    if kind == 1:
        return np.sort(rng.integers(-10, total + 11, batch + 1))
    if kind == 2:
        return rng.integers(-10, total + 11, batch + 1)
    return rng.choice([LOWEST, LOWEST + 1, -1, 0, total // 2, total, HIGHEST], batch + 1)


def bits(rng, *shape):
    return O.f32_to_bf16(rng.standard_normal(shape).astype(np.float32))


def main(path, seed):
    lib = ctypes.CDLL(path)
    lib.model_seed(seed)
    rng = np.random.default_rng(seed)
    f64 = lambda b: O.bf16_to_f32(b).astype(np.float64)  # noqa: E731
    for i in range(12):
        batch, total, slots = int(rng.integers(1, 6)), int(rng.integers(1, 40)), int(rng.integers(1, 5))
        starts = starts_of(rng, batch, total).astype(np.int32)
        read = rng.choice([LOWEST, -1, 0, slots - 1, slots, HIGHEST], batch).astype(np.int32)
        # (a slot that one sequence writes is read by that one only)
        cols = int(rng.choice([0, 0, 1, 3]))
        write = rng.choice([LOWEST, -1, slots, HIGHEST], (batch, max(cols, 1))).astype(np.int32)
        own = int(rng.integers(batch))
        write[own, 0] = 0
        read[(read == 0) & (np.arange(batch) != own)] = -1
        ordered = (np.diff(starts.astype(np.int64)) >= 0).all()
        lens = np.diff(np.clip(starts, 0, total)) if ordered else None
        at, at_end = int(np.clip(starts[0], 0, total)), bool(rng.integers(2))
        held = [guarded(a, at_end) for a in (starts, read, write)]
        sizes = (total, batch, int(rng.choice([0, 1, total, 100])), slots, cols)
        of = lambda *g: [ctypes.c_void_p(None if x is None else x.at) for x in g]  # noqa: E731

        C, W = 16, int(rng.integers(2, 5))
        x, w, state = bits(rng, total, C), bits(rng, C, W), bits(rng, slots, W - 1, C)
        g = [guarded(a, at_end) for a in (x, w, state)]
        out = Guarded(2 * total * C)
        lib.model_conv(*of(*g, *held, out), *sizes, C, W)
        if ordered:
            with np.errstate(invalid="ignore"):
                ref, tol, _ = DO.conv(f64(x)[at:at + lens.sum()], f64(w), None, f64(state), lens, read)
            got = f64(out.array(np.uint16).reshape(total, C))[at:at + lens.sum()]
            fine = np.isfinite(ref)
            assert (np.isfinite(got) == fine).all() and (np.abs(got - ref)[fine] <= tol[fine]).all(), i

        Hk, Hv, d = 1, 2, 64
        q, k, v = bits(rng, total, Hk, d), bits(rng, total, Hk, d), bits(rng, total, Hv, d)
        a, b = bits(rng, total, Hv), bits(rng, total, Hv)
        a_log, dt = np.zeros(Hv, np.float32), np.full(Hv, -2, np.float32)
        state = rng.standard_normal((slots, Hv, d, d)).astype(np.float32)
        g = [guarded(t, at_end) for t in (q, k, v, a, b, a_log, dt, state)]
        out = Guarded(2 * total * Hv * d)
        lib.model_steps(*of(*g, *held, out), *sizes, Hk, Hv)
        if ordered:
            n = slice(at, at + lens.sum())
            ref, tol, *_ = DO.delta(f64(q)[n], f64(k)[n], f64(v)[n], f64(a)[n], f64(b)[n], a_log.astype(float),
                                    dt.astype(float), state.astype(float), lens, read)
            got = f64(out.array(np.uint16).reshape(total, Hv, d))[n]
            fine = np.isfinite(ref)
            assert (np.isfinite(got) == fine).all() and (np.abs(got - ref)[fine] <= tol[fine]).all(), i
    print(f"seed {seed}", flush=True)


if __name__ == "__main__":
    main(sys.argv[1], int(sys.argv[2]))
