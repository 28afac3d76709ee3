"""One token of each row of logits (gfx950), by temperature, top-k, top-p and min-p, from given uniform
random numbers.

The HIP library does the work; there is no torch fallback. A call runs on the current stream of its
tensors' device and allocates through torch only, so it can be captured into a graph. What the host can see
is checked before anything is launched (RuntimeError). The same inputs always give the same tokens.

Op: radiance::sample, with a fake, opaque to a compiler.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native_decode as _native
from .radiance_kv4 import _entry


def _sample(logits: torch.Tensor, uniform: torch.Tensor, temperature: Optional[torch.Tensor],
            top_k: Optional[torch.Tensor], top_p: Optional[torch.Tensor], min_p: Optional[torch.Tensor],
            temperature_all: float, top_k_all: int, top_p_all: float, min_p_all: float,
            logprobs: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return _native.ops().sample(logits, uniform, temperature, top_k, top_p, min_p, temperature_all,
                                top_k_all, top_p_all, min_p_all, logprobs)


def _sample_fake(logits, uniform, temperature, top_k, top_p, min_p, temperature_all, top_k_all, top_p_all,
                 min_p_all, logprobs):
    rows = logits.shape[0]
    return (torch.empty(rows, dtype=torch.int64, device=logits.device),
            torch.empty(rows if logprobs else 0, dtype=torch.float32, device=logits.device))


sample_op = torch.library.custom_op("radiance::sample", _sample, mutates_args=())
sample_op.register_fake(_sample_fake)
_call_sample = _entry(sample_op, "sample", _native)


def _per_row(x, default):
    """A parameter as (tensor or None, the value for all rows)."""
    if x is None:
        return None, default
    return (x, default) if isinstance(x, torch.Tensor) else (None, type(default)(x))


def sample(logits, uniform, *, temperature=1.0, top_k=None, top_p=None, min_p=None, logprobs: bool = False):
    """The tokens int64 [rows] of logits fp32 or bf16 [rows, vocabulary], and with `logprobs` their log
    probabilities fp32 [rows] under the softmax of the logits as they are (no temperature, no filter).

    Weights are exp((x - max) / temperature). Of the row in descending order, ties by index, the first top_k
    stay; of those the shortest prefix with at least top_p of their weight; of those the ones whose weight
    is at least min_p times the largest. The token is the lowest index at which the sum of what stays, up
    to it, exceeds uniform (fp32 [rows], in [0, 1)) times their sum. Each parameter is a number or a tensor
    for the rows (temperature, top_p, min_p fp32, top_k int32 [rows]; numbers have these ranges too); None or
    a value outside of what filters filters nothing, temperature 0 takes the first of the largest. A row that holds NaN, or nothing above
    -infinity, gives -1 (log probability NaN). Weights are added as whole numbers of 2^-min(51, 62 -
    ceil(log2 vocabulary)), so that no order of additions changes a token; one of less than half of that is
    none."""
    t, t_all = _per_row(temperature, 1.0)
    k, k_all = _per_row(top_k, 0)
    p, p_all = _per_row(top_p, 1.0)
    mp, mp_all = _per_row(min_p, 0.0)
    tokens, lp = _call_sample(logits, uniform, t, k, p, mp, t_all, k_all, p_all, mp_all, bool(logprobs))
    return (tokens, lp) if logprobs else tokens
