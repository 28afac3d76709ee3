"""Definitions in 64 bits of the operators of include/decode_ops.h, in numpy, with the error bounds that the
tests hold the kernels to."""
import numpy as np

EPS32 = 2.0 ** -24              # half a step of fp32
EPSBF = 2.0 ** -8               # half a step of bf16


def silu(x):
    return x / (1 + np.exp(-x))


def conv(x, weight, bias, state, lens, read, silu_=True):
    """x [T, C], weight [C, W], bias [C] or None, state [slots, W - 1, C], all float64. Returns (out [T, C], the
    bound on a kernel's error, and for each sequence the inputs from its state on, [W - 1 + n, C])."""
    W = weight.shape[1]
    out, tol, seen, at = np.empty_like(x), np.empty_like(x), [], 0
    for b, n in enumerate(lens):
        r = read[b]
        past = np.zeros_like(state[0]) if r < 0 else np.full_like(state[0], np.nan) if r >= len(state) else state[r]
        y = np.concatenate([past, x[at:at + n]])
        terms = [weight[:, i] * y[i:i + n] for i in range(W)]
        z = sum(terms) + (0 if bias is None else bias)
        size = sum(np.abs(t) for t in terms) + (0 if bias is None else np.abs(bias))
        with np.errstate(over="ignore", invalid="ignore"):
            o = silu(z) if silu_ else z
        out[at:at + n] = o
        # W fused additions in fp32; SiLU's slope is below 1.1, its exponential, sum and quotient are each
        # within 4 steps; one rounding to bf16
        slack = 1.1 * W * EPS32 * size + 12 * EPS32 * np.abs(o)
        tol[at:at + n] = EPSBF * (np.abs(o) + slack) + slack + 2.0 ** -126
        seen.append(y)
        at += n
    return out, tol, seen


def gates(a, b, a_log, dt_bias):
    """Log decay and beta [T, H]."""
    x = a + dt_bias
    with np.errstate(over="ignore"):
        return -np.exp(a_log) * np.logaddexp(x, 0), 1 / (1 + np.exp(-b))


def delta(q, k, v, a, b, a_log, dt_bias, state, lens, read, scale=None, eps=1e-6):
    """All float64; q, k [T, Hk, dk], v [T, Hv, dv], state [slots, Hv, dk, dv]. Returns (out [T, Hv, dv], bound,
    and for each sequence its states from the initial one on [n + 1, Hv, dk, dv] with their bounds
    [n + 1, Hv, dv] for the 2-norm of a column's error).

    The bound follows the columns' errors: a step maps a column's error with e^g (1 - beta k k^T), which is no
    longer than e^g, and adds what its own operations round. Those are sums of dk terms and a few more
    operations in fp32, in whatever order, of columns no longer than |S|, |u| and |v|: 2 dk + 64 roundings. The
    exponential of a chunk's sum of log decays is off by the rounding of each one's, |g| of 8 steps."""
    T, Hk, dk = q.shape
    Hv, dv = v.shape[1:]
    scale = dk ** -0.5 if scale is None else scale
    g, beta = gates(a, b, a_log, dt_bias)
    unit = lambda x: x / np.sqrt((x * x).sum(-1, keepdims=True) + eps)  # noqa: E731
    q, k = (np.repeat(unit(x), Hv // Hk, 1) for x in (q, k))
    out, tol = np.empty((T, Hv, dv)), np.empty((T, Hv, dv))
    states, bounds, at = [], [], 0
    c = (2 * dk + 64) * EPS32
    for i, n in enumerate(lens):
        r = read[i]
        S = np.zeros(state.shape[1:]) if r < 0 else np.full(state.shape[1:], np.nan) if r >= len(state) else state[r]
        E = np.zeros((Hv, dv))
        ss, es = [S], [E]
        for t in range(at, at + n):
            alpha = np.exp(g[t])[:, None]
            before = np.sqrt((S * S).sum(1))
            S = alpha[..., None] * S
            u = beta[t][:, None] * (v[t] - (S * k[t][..., None]).sum(1))
            S = S + k[t][..., None] * u[:, None]
            size = before + np.abs(u) + np.abs(v[t])
            slip = 8 * EPS32 * np.minimum(-g[t], 100.0)[:, None] * alpha * before
            E = alpha * E + c * size + slip
            o = scale * (S * q[t][..., None]).sum(1)
            out[t] = o
            slack = abs(scale) * (E + c * (size + np.sqrt((S * S).sum(1))))
            tol[t] = EPSBF * (np.abs(o) + slack) + slack + 2.0 ** -126
            ss.append(S), es.append(E)
        states.append(np.stack(ss)), bounds.append(np.stack(es))
        at += n
    return out, tol, states, bounds


def order_of(x):
    """Indices of a row in descending order, ties by index."""
    return np.lexsort((np.arange(len(x)), -x))


def sample(x, u, t=1.0, k=0, p=1.0, mp=0.0):
    """(token, log probability) of a row x of logits."""
    x = np.asarray(x, np.float64)
    if np.isnan(x).any() or x.max() == -np.inf or np.isnan(t):
        return -1, np.nan
    top = x.max()
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        z = np.where(x == top, 0.0, x - top)
        lp = z - np.log(np.exp(z).sum())
        order = order_of(x)
        if not t > 0:
            return int(order[0]), lp[order[0]]
        w = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.exp(z / t)))
    if 1 <= k < len(x):
        order = order[:k]
    if p < 1:
        mass = np.cumsum(w[order])
        order = order[:1 + int(np.searchsorted(mass, p * mass[-1]))] if p > 0 else order[:1]
    if mp > 0:
        order = order[np.maximum(w[order] >= mp, np.arange(len(order)) == 0)]
    order = np.sort(order)
    mass = np.cumsum(w[order])
    u = 0.0 if np.isnan(u) else min(max(u, 0.0), 1.0)
    at = int(np.searchsorted(mass, u * mass[-1], side="right"))
    if at >= len(order):                # u at 1: the last of any weight
        at = int(np.nonzero(w[order] > 0)[0][-1])
    return int(order[at]), lp[order[at]]
