"""Attention over a paged key/value cache held in 4 bits (gfx950): what lies between a decoder's qkv
and output projections (radiance_mxfp4 has those).

  qk_norm_rope         per-head RMSNorm of queries and keys with the rotation, one to several axes
  qk_norm_rope_append  the same, with the new keys and values rounded into their cache slots
  attention            softmax attention of ragged queries over the cached tokens
  gather               tokens of the cache as bf16
  move_pages           page copies over all layers, and the remapped page table, in one launch

kv4_pool.PagePool is the host's side: allocate, extend, fork, truncate, free, compact.

The cache is MXFP4, as the weights are: e2m1 codes with a power-of-two scale for each 32 channels of a
token, 4.25 bits an element. new_cache() makes one: uint8 [pages, kv heads, page / 16, 17 d], or
with a leading axis of layers. Head sizes 64, 128, 256; pages of 16, 32, 64, 128 or 256 tokens. The bytes
of a group of 16 tokens are laid out in matrix-operand order (include/kv4_attn.h). A slot is page
number * page + place.

The HIP library does the work; there is no torch fallback. Every call runs on the current stream of
its tensors' device and allocates through torch only, so it can be captured into a graph. What the
host can see is checked before anything is launched (RuntimeError); what only the device knows is
checked there: a position outside the table or a page outside the cache gives NaN, a slot outside
the cache is not written. Inference only: no op here has a gradient.

Ops: radiance::qk_norm_rope, ::qk_norm_rope_kv4, ::kv4_attention, ::kv4_gather, ::kv4_move_pages, each
with a fake, opaque to a compiler. The functions are the same with defaults.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import _native_kv4 as _native
from . import radiance_mxfp4 as _rmx

HEAD_SIZES = (64, 128, 256)
PAGE_SIZES = (16, 32, 64, 128, 256)
GROUP = 16                      # tokens of a group


def _fail(op: str, what: str):
    raise RuntimeError(f"[radiance.kv4] {op}: {what}")


def new_cache(pages: int, kv_heads: int, page: int, head_size: int, device="cuda",
              layers: Optional[int] = None) -> torch.Tensor:
    """An empty cache (every token reads as zero): uint8 [pages, kv_heads, page / 16, 17 * head_size],
    with `layers` a leading axis of that many. A layer's cache is cache[layer]."""
    if head_size not in HEAD_SIZES or page not in PAGE_SIZES:
        _fail("new_cache", f"head size {head_size} is none of {HEAD_SIZES} or page {page} none of "
                           f"{PAGE_SIZES}")
    shape = (pages, kv_heads, page // GROUP, 17 * head_size)
    return torch.zeros(shape if layers is None else (layers, *shape), dtype=torch.uint8,
                       device=device)


def rotary_axes(sections: Sequence[int], interleaved: bool = False, device="cuda") -> torch.Tensor:
    """The axis of each rotated pair, int32 [sum(sections)], for `axis` of the norm-and-rotate ops:
    sections[a] pairs turn by the position on axis a, all of axis 0 first, then axis 1 and so on; or
    interleaved: pair p takes axis p % axes while that axis has pairs left, else axis 0."""
    sections = [int(s) for s in sections]
    n, total = len(sections), sum(sections)
    if not sections or min(sections) < 0 or total == 0:
        _fail("rotary_axes", f"sections {sections}")
    if interleaved:
        axes = [p % n if p // n < sections[p % n] else 0 for p in range(total)]
        if [axes.count(a) for a in range(n)] != sections:
            _fail("rotary_axes", f"sections {sections} cannot be interleaved")
    else:
        axes = [a for a, s in enumerate(sections) for _ in range(s)]
    return torch.tensor(axes, dtype=torch.int32, device=device)


_compiling, _jit_tracing = _rmx._compiling, _rmx._jit_tracing
_dispatch_modes, _function_modes = _rmx._dispatch_modes, _rmx._function_modes


def _entry(op, name):
    """The native op `name`, called without the dispatcher (3 us a call) where nothing watches ops by name
    and every tensor is plain; else `op`, whose name a compiler, a tracer, a mode or a subclass sees, which
    vmap maps and whose backward raises. The binding looks at the tensors (kv4_torch.cpp), 1 us a call less
    than fewer of these checks took here."""
    ns, public = op._qualname.split("::")
    space = getattr(torch.ops, ns)
    name += "_if_plain"

    def call(*args):
        # _rmx._watched() inline, as in its own call sites
        if not (_compiling() or _dispatch_modes() or _jit_tracing()
                or (_function_modes() and _rmx._function_mode_watches())):
            out = getattr(_native.ops(), name)(*args)
            if out is not NotImplemented:
                return out
        return getattr(space, public)(*args)
    return call


# ---- norm and rotation --------------------------------------------------------------------------
def _qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor],
                  k_weight: Optional[torch.Tensor], cos_sin: Optional[torch.Tensor],
                  positions: Optional[torch.Tensor], axis: Optional[torch.Tensor], eps: float,
                  plus_one: bool, adjacent: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return _native.ops().qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, axis, eps,
                                      plus_one, adjacent)


def _qk_norm_rope_fake(q, k, q_weight, k_weight, cos_sin, positions, axis, eps, plus_one, adjacent):
    return (torch.empty(q.shape, dtype=torch.bfloat16, device=q.device),
            torch.empty(k.shape, dtype=torch.bfloat16, device=k.device))


qk_norm_rope_op = torch.library.custom_op("radiance::qk_norm_rope", _qk_norm_rope, mutates_args=())
qk_norm_rope_op.register_fake(_qk_norm_rope_fake)
_call_qk_norm_rope = _entry(qk_norm_rope_op, "qk_norm_rope")


def qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, *, axis=None, eps: float = 1e-6,
                 plus_one: bool = False, adjacent: bool = False):
    """RMSNorm of each head of q [T, q heads, d] and k [T, kv heads, d] (bf16, views of a wider
    projection as they are) with the weights bf16 [d] (plus_one: w + 1; None: no norm), then the
    rotation: cos_sin [positions, rot] holds rot / 2 cosines and as many sines (fp32 or bf16; None: no
    rotation), pairs are (p, p + rot / 2), or (2p, 2p + 1) with adjacent, and channels from rot on stay.
    positions int64 or int32 [T], or [axes, T] with axis = rotary_axes(sections). Computed in fp32 and
    rounded once. Returns (q, k), new and contiguous."""
    return _call_qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, axis, float(eps),
                              bool(plus_one), bool(adjacent))


def _qk_norm_rope_kv4(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                      cos_sin: Optional[torch.Tensor], positions: Optional[torch.Tensor],
                      cache: torch.Tensor, slots: torch.Tensor, axis: Optional[torch.Tensor],
                      eps: float, plus_one: bool, adjacent: bool) -> torch.Tensor:
    return _native.ops().qk_norm_rope_append(q, k, v, q_weight, k_weight, cos_sin, positions, cache,
                                             slots, axis, eps, plus_one, adjacent)


def _qk_norm_rope_kv4_fake(q, k, v, q_weight, k_weight, cos_sin, positions, cache, slots, axis, eps,
                           plus_one, adjacent):
    return torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)


qk_norm_rope_kv4_op = torch.library.custom_op("radiance::qk_norm_rope_kv4", _qk_norm_rope_kv4,
                                              mutates_args=("cache",))
qk_norm_rope_kv4_op.register_fake(_qk_norm_rope_kv4_fake)
_call_qk_norm_rope_kv4 = _entry(qk_norm_rope_kv4_op, "qk_norm_rope_append")


def qk_norm_rope_append(q, k, v, q_weight, k_weight, cos_sin, positions, cache, slots, *, axis=None,
                        eps: float = 1e-6, plus_one: bool = False, adjacent: bool = False):
    """qk_norm_rope, with the keys (rounded from fp32) and the values v [T, kv heads, d] written into
    `cache` at `slots` (int64 [T], distinct; negative ones are skipped, for padding). Returns q."""
    return _call_qk_norm_rope_kv4(q, k, v, q_weight, k_weight, cos_sin, positions, cache, slots, axis,
                                  float(eps), bool(plus_one), bool(adjacent))


# ---- reading back -------------------------------------------------------------------------------
def _kv4_gather(cache: torch.Tensor, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return _native.ops().gather(cache, slots)


def _kv4_gather_fake(cache, slots):
    shape = (slots.shape[0], cache.shape[1], cache.shape[3] // 17)
    return (torch.empty(shape, dtype=torch.bfloat16, device=cache.device),
            torch.empty(shape, dtype=torch.bfloat16, device=cache.device))


kv4_gather_op = torch.library.custom_op("radiance::kv4_gather", _kv4_gather, mutates_args=())
kv4_gather_op.register_fake(_kv4_gather_fake)
_call_kv4_gather = _entry(kv4_gather_op, "gather")


def gather(cache, slots):
    """The keys and values at `slots` (int64 [T]) as bf16 [T, kv heads, d], exactly what the cache
    holds; zeros at a negative slot, NaN at one past the cache."""
    return _call_kv4_gather(cache, slots)


# ---- attention ----------------------------------------------------------------------------------
def _kv4_attention(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor,
                   seq_lens: torch.Tensor, q_starts: torch.Tensor, max_q: int, max_len: int,
                   scale: float, causal: bool, window: int) -> torch.Tensor:
    return _native.ops().attention(q, cache, page_table, seq_lens, q_starts, max_q, max_len, scale,
                                   causal, window)


def _kv4_attention_fake(q, cache, page_table, seq_lens, q_starts, max_q, max_len, scale, causal,
                        window):
    return torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)


kv4_attention_op = torch.library.custom_op("radiance::kv4_attention", _kv4_attention,
                                           mutates_args=())
kv4_attention_op.register_fake(_kv4_attention_fake)
_call_kv4_attention = _entry(kv4_attention_op, "attention")


def attention(q, cache, page_table, seq_lens, q_starts, max_q: int, max_len: int, *,
              scale: Optional[float] = None, causal: bool = True, window: int = 0):
    """Softmax attention over the cached tokens. q bf16 [total, q heads, d]; sequence b's queries
    are rows q_starts[b] .. q_starts[b + 1] - 1 (int32 [batch + 1]) and are the last of its seq_lens[b]
    cached tokens (int32 [batch]; append them first); its pages are page_table[b] (int32
    [batch, ...]), in order. max_q and max_len: at least the most queries and tokens of a sequence;
    they size the launch, so a graph captured with a batch's limits serves any lengths within them.
    scale: 1 / sqrt(d) by default. causal: a query sees its own place and those before it; window > 0:
    the last `window` of those; a query that sees none gives zeros. Query heads share kv heads in
    consecutive groups. Returns bf16 [total, q heads, d]; rows that no sequence owns are not
    written."""
    return _call_kv4_attention(q, cache, page_table, seq_lens, q_starts, int(max_q), int(max_len),
                               float(1.0 / math.sqrt(q.shape[-1]) if scale is None else scale),
                               bool(causal), int(window))


# ---- pages --------------------------------------------------------------------------------------
def _kv4_move_pages(cache: torch.Tensor, pairs: torch.Tensor,
                    page_table: Optional[torch.Tensor]) -> None:
    return _native.ops().move_pages(cache, pairs, page_table)


def _kv4_move_pages_fake(cache, pairs, page_table):
    return None


kv4_move_pages_op = torch.library.custom_op("radiance::kv4_move_pages", _kv4_move_pages,
                                            mutates_args=("cache", "page_table"))
kv4_move_pages_op.register_fake(_kv4_move_pages_fake)
_call_kv4_move_pages = _entry(kv4_move_pages_op, "move_pages")


def move_pages(cache, pairs, page_table=None) -> None:
    """Copies page pairs[i, 0] to page pairs[i, 1] (int32 [n, 2] on the host, read before the call
    returns) in a layer's cache or in all layers of one, and replaces the first by the second in
    page_table (int32 [sequences, pages], contiguous rows) where one is given. One launch per 448
    pairs. Refused: a page both read and written, a page written twice and, with a table, a page read
    twice."""
    _call_kv4_move_pages(cache, pairs, page_table)
