"""What lies between the in- and output projections of a linear-attention (gated delta net) layer
(gfx950); radiance_fused_norm.gdn_norm_quant, the gated norm in front of the output projection, comes
after it.

  causal_conv         the short convolution over the channels of q, k and v, with SiLU
  gated_delta_rule    the gated delta rule over the batch's sequences: prompts in chunks, decoded and
                      drafted tokens one by one

Both go on from a state for each sequence and leave the new one: new_conv_state and new_state make pools of
slots, and a call says for each sequence of its batch which slot it reads (negative: it begins from zeros) and
which it writes. The same slot is the usual step; another one forks a sequence; and with a slot for each token
(write_slots [batch, tokens]) the state after every drafted token is kept, so that the next call reads
that of the last one accepted. A slot that one sequence writes may be read by no other in the call, and
written by no other.

A batch's tokens lie one sequence after the other, q_starts as in radiance_kv4.attention; PagePool's steps
have them. max_q, at least the most tokens of a sequence, chooses how the work is done, not what comes out (the
delta rule's two forms round differently): a graph captured with it serves any starts and slots. With max_q above 16 all
sequences of a call go in chunks of 64 tokens, also those of one; decoding sequences beside a prompt are better a
call of their own. Chunks take a workspace while the call runs (include/decode_ops.h has its size).

The HIP library does the work; there is no torch fallback. Every call runs on the current stream of its
tensors' device and allocates through torch only, so it can be captured into a graph. What the host can
see is checked before anything is launched (RuntimeError); what only the device knows is checked there: a
sequence that reads a slot past the pool gives NaN, a slot outside the pool is not written. Inference only:
no op here has a gradient.

Ops: radiance::causal_conv, ::gated_delta_rule, each with a fake, opaque to a compiler. The functions are the
same with defaults.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native_decode as _native
from .radiance_kv4 import _entry

HEAD_SIZES = (64, 128)
WIDTHS = (2, 3, 4)


def _fail(op: str, what: str):
    raise RuntimeError(f"[radiance.decode] {op}: {what}")


def new_state(slots: int, v_heads: int, k_size: int, v_size: int, device="cuda",
              layers: Optional[int] = None) -> torch.Tensor:
    """States of the delta rule, all zeros: fp32 [slots, v_heads, k_size, v_size], with `layers` a leading
    axis of that many. A layer's is state[layer]."""
    if k_size not in HEAD_SIZES or v_size not in HEAD_SIZES:
        _fail("new_state", f"heads of {k_size} and {v_size} channels are none of {HEAD_SIZES}")
    shape = (slots, v_heads, k_size, v_size)
    return torch.zeros(shape if layers is None else (layers, *shape), dtype=torch.float32, device=device)


def new_conv_state(slots: int, channels: int, width: int, device="cuda",
                   layers: Optional[int] = None) -> torch.Tensor:
    """States of the convolution, all zeros: bf16 [slots, width - 1, channels], the last inputs of a
    sequence, oldest first; with `layers` a leading axis of that many."""
    if width not in WIDTHS or channels % 8:
        _fail("new_conv_state", f"width {width} is none of {WIDTHS}, or {channels} channels no multiple of 8")
    shape = (slots, width - 1, channels)
    return torch.zeros(shape if layers is None else (layers, *shape), dtype=torch.bfloat16, device=device)


# ---- convolution --------------------------------------------------------------------------------
def _causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], state: torch.Tensor,
                 q_starts: torch.Tensor, read_slots: torch.Tensor, write_slots: torch.Tensor, max_q: int,
                 silu: bool) -> torch.Tensor:
    return _native.ops().causal_conv(x, weight, bias, state, q_starts, read_slots, write_slots, max_q, silu)


def _causal_conv_fake(x, weight, bias, state, q_starts, read_slots, write_slots, max_q, silu):
    return torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)


causal_conv_op = torch.library.custom_op("radiance::causal_conv", _causal_conv, mutates_args=("state",))
causal_conv_op.register_fake(_causal_conv_fake)
_call_causal_conv = _entry(causal_conv_op, "causal_conv", _native)


def causal_conv(x, weight, bias, state, q_starts, read_slots, write_slots, max_q: int, *, silu: bool = True):
    """out[t, c] = silu(bias[c] + sum_i weight[c, i] x[t - width + 1 + i, c]) over each sequence's tokens,
    x bf16 [total, channels] (a view of a wider projection as it is), weight bf16 [channels, width] (width 2,
    3 or 4), bias bf16 [channels] or None, state as new_conv_state makes it. Sequence b's tokens are rows
    q_starts[b] .. q_starts[b + 1] - 1 (int32 [batch + 1]); before them come the inputs in slot
    read_slots[b] (int32 [batch]); write_slots int32 [batch] (after the last token) or [batch, tokens] (after
    each). Computed in fp32 and rounded once. Returns bf16 [total, channels]; rows that no sequence owns are
    not written."""
    return _call_causal_conv(x, weight, bias, state, q_starts, read_slots, write_slots, int(max_q), bool(silu))


# ---- gated delta rule ---------------------------------------------------------------------------
def _gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                      a_log: torch.Tensor, dt_bias: torch.Tensor, state: torch.Tensor,
                      q_starts: torch.Tensor, read_slots: torch.Tensor, write_slots: torch.Tensor,
                      max_q: int, scale: Optional[float], eps: float) -> torch.Tensor:
    return _native.ops().gated_delta_rule(q, k, v, a, b, a_log, dt_bias, state, q_starts, read_slots,
                                          write_slots, max_q, scale, eps)


def _gated_delta_rule_fake(q, k, v, a, b, a_log, dt_bias, state, q_starts, read_slots, write_slots, max_q,
                           scale, eps):
    return torch.empty(v.shape, dtype=torch.bfloat16, device=v.device)


gated_delta_rule_op = torch.library.custom_op("radiance::gated_delta_rule", _gated_delta_rule,
                                              mutates_args=("state",))
gated_delta_rule_op.register_fake(_gated_delta_rule_fake)
_call_gated_delta_rule = _entry(gated_delta_rule_op, "gated_delta_rule", _native)


def gated_delta_rule(q, k, v, a, b, a_log, dt_bias, state, q_starts, read_slots, write_slots, max_q: int, *,
                     scale: Optional[float] = None, eps: float = 1e-6):
    """For each sequence and value head, with the state S [key channels, value channels] in fp32, token after
    token: S <- e^g S; u = beta (v - S^T k); S <- S + k u^T; out = scale S^T q, where q and k are
    divided by sqrt(sum of squares + eps), g = -exp(a_log) softplus(a + dt_bias), beta = sigmoid(b).

    q, k bf16 [total, key heads, 64 or 128] and v bf16 [total, value heads, 64 or 128], views of the
    convolution's output as they are; value heads share key heads in consecutive groups. a, b bf16 [total,
    value heads]; a_log, dt_bias fp32 [value heads]. scale: 1 / sqrt(key channels) by default. state as
    new_state makes it; starts and slots as for causal_conv. Returns bf16 [total, value heads, channels];
    rows that no sequence owns are not written."""
    return _call_gated_delta_rule(q, k, v, a, b, a_log, dt_bias, state, q_starts, read_slots, write_slots,
                                  int(max_q), None if scale is None else float(scale), float(eps))
