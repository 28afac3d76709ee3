"""Runs the sampling kernels, compiled for the CPU (tests/test_cpu_model.py), over cases of one seed and compares the tokens
with the definition's. Logits, parameters, outputs and workspace each end, or begin, at memory that cannot be touched.

  python -m tests.cpu_model.sample LIBRARY SEED
"""
import ctypes
import sys

import numpy as np

from oracle import decode_oracle as DO
from oracle import mxfp4_oracle as O
from tests.cpu_model.memory import Guarded, guarded


class Args(ctypes.Structure):
    """dec::SampleArgs (dec_internal.h)."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("logits", "uniform", "temperature", "top_k", "top_p", "min_p", "tokens",
                                                "logprobs", "workspace")]
                + [("row_stride", ctypes.c_long)] + [(n, ctypes.c_int) for n in ("rows", "V", "top_k_all", "parts")]
                + [(n, ctypes.c_float) for n in ("temperature_all", "top_p_all", "min_p_all")]
                + [("bf16", ctypes.c_bool)])


def check(lib, x, u, parts, at_end, bf16=False, t=None, k=None, p=None, mp=None, k_all=0):
    rows, V = x.shape
    f = np.float32
    held = [guarded(x, at_end)] + [guarded(None if a is None else np.asarray(a, d), at_end)
                                   for a, d in ((u, f), (t, f), (k, np.int32), (p, f), (mp, f))]
    tokens, logprobs = Guarded(8 * rows), Guarded(4 * rows)
    space = Guarded(lib.model_workspace(rows, parts), True, 16)
    a = Args(*[None if h is None else h.at for h in held], tokens.at, logprobs.at, space.at, V, rows, V, k_all, parts,
             1.0, 1.0, 0.0, bf16)
    assert lib.model_args() == ctypes.sizeof(Args)
    assert lib.model_sample(ctypes.byref(a)) == 0
    values = O.bf16_to_f32(x) if bf16 else x
    of = lambda a, i, d: d if a is None else float(f(a[i]))  # noqa: E731
    for i in range(rows):
        how = of(t, i, 1.0), int(k[i]) if k is not None else k_all, of(p, i, 1.0), of(mp, i, 0.0)
        want, lp = DO.sample(values[i], float(f(u[i])), *how)
        got, got_lp = int(tokens.array(np.int64)[i]), float(logprobs.array(f)[i])
        assert got == want, (parts, i, got, want, how)
        assert np.isnan(lp) and np.isnan(got_lp) or got_lp == lp or abs(got_lp - lp) < 1e-4, (parts, i, got_lp, lp)


def main(path, seed):
    lib = ctypes.CDLL(path)
    lib.model_workspace.restype = ctypes.c_size_t
    lib.model_seed(seed)
    rng = np.random.default_rng(seed)
    rows = 2
    sizes = (1, 2, 63, 1500, 2049, 5000, 9000, 13001)
    V = sizes[seed % len(sizes)]
    x = (rng.uniform(0.5, 4) * rng.standard_normal((rows, V))).astype(np.float32)
    kind = seed // 2 % 5 if V > 70 else 0
    if kind == 1:
        x = np.round(x)                                 # ties
    if kind == 2:
        x[0] = 0.25
    if kind == 3:
        x = np.where(rng.random((rows, V)) < 0.99, -np.inf, x).astype(np.float32)
        x[:, 5] = 1
    if kind == 4:
        x[0, 3], x[1, [7, 70]] = np.nan, np.inf
    bf16 = bool(seed % 2)
    if bf16:
        x = O.f32_to_bf16(x)
    u, t = rng.random(rows), rng.uniform(0.3, 1.5, rows)
    k, p, mp = rng.integers(1, 400, rows), rng.uniform(0.2, 1.1, rows), rng.uniform(-0.05, 0.2, rows)
    cases = [(dict(t=t), 1), (dict(t=t, k=k, p=p, mp=mp), 1), (dict(p=p), 1), (dict(p=[0.6, 0.999999], t=[0.01, 50]), 3),
             (dict(k_all=700, p=p, mp=mp), 2), (dict(t=[0.0, 0.02]), 5), (dict(k=[513, 3000], p=p), 1)]
    for i, (kw, parts) in enumerate(cases):
        check(lib, x, u, parts, (seed + i) % 2 == 0, bf16, **kw)
    print(f"seed {seed}: {len(cases)} calls of {rows} rows of {V}", flush=True)


if __name__ == "__main__":
    main(sys.argv[1], int(sys.argv[2]))
