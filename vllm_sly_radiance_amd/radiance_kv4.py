"""Attention over a paged key/value cache held in 4 bits (gfx950): what lies between a decoder's qkv
and output projections (radiance_mxfp4 has those).

  qk_norm_rope         per-head RMSNorm of queries and keys with the rotation, one to several axes
  qk_norm_rope_append  the same, with the new keys and values rounded into their cache slots
  attention            softmax attention of ragged queries over the cached tokens
  gather               tokens of the cache as bf16
  move_pages           page copies over all layers, and the remapped page table, in one launch
  PagePool             the host's side: allocate, extend, fork, free, compact

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


# ---- checks -------------------------------------------------------------------------------------
def _heads(op: str, name: str, x: torch.Tensor) -> torch.Tensor:
    """bf16 [T, heads, d] whose heads are 16-byte aligned runs; other layouts are copied."""
    if x.dtype != torch.bfloat16 or x.dim() != 3:
        _fail(op, f"{name} must be bf16 [tokens, heads, head size], got {x.dtype} {tuple(x.shape)}")
    if x.shape[2] not in HEAD_SIZES:
        _fail(op, f"head size {x.shape[2]} of {name} is none of {HEAD_SIZES}")
    if x.shape[0] == 0:
        return x
    st, sh, sc = x.stride()
    if sc != 1 or x.data_ptr() % 16 or (st % 8 and x.shape[0] > 1) or (sh % 8 and x.shape[1] > 1) \
            or st < 0 or sh < 0:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _strides(x: torch.Tensor):
    """Token and head strides; those of an axis of one, which may be anything, as 0."""
    return (x.stride(0) if x.shape[0] > 1 else 0), (x.stride(1) if x.shape[1] > 1 else 0)


def _cache(op: str, cache: torch.Tensor, d: Optional[int] = None, heads: Optional[int] = None):
    """(page size, page stride) of a layer's cache."""
    if cache.dtype != torch.uint8 or cache.dim() != 4 or cache.shape[3] % 17 \
            or cache.shape[3] // 17 not in HEAD_SIZES or cache.shape[2] * GROUP not in PAGE_SIZES:
        _fail(op, f"cache must be uint8 [pages, kv heads, page / 16, 17 * head size], got "
                  f"{cache.dtype} {tuple(cache.shape)}")
    _, H, n, b = cache.shape
    if cache.numel() and ((H > 1 and cache.stride(1) != n * b) or (n > 1 and cache.stride(2) != b)
                          or cache.stride(3) != 1 or cache.data_ptr() % 16):
        _fail(op, "a page of the cache must be contiguous and 16-byte aligned")
    if d is not None and b != 17 * d:
        _fail(op, f"cache of head size {b // 17} against {d}")
    if heads is not None and H != heads:
        _fail(op, f"cache of {H} kv heads against {heads}")
    return n * GROUP, (cache.stride(0) if cache.shape[0] > 1 else H * n * b)


def _same_device(op: str, *tensors):
    dev = tensors[0].device
    if dev.type != "cuda":
        _fail(op, f"tensors must be on the GPU, got {dev}")
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            _fail(op, f"tensors on {dev} and {t.device}")
    return dev


class _on:
    """The tensors' device as the current one, where it is not already."""

    def __init__(self, dev):
        self.other = None if dev.index is None or dev.index == torch.cuda.current_device() \
            else torch.cuda.device(dev)

    def __enter__(self):
        if self.other is not None:
            self.other.__enter__()

    def __exit__(self, *exc):
        if self.other is not None:
            self.other.__exit__(*exc)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _slots(op: str, slots: torch.Tensor, T: int) -> torch.Tensor:
    if slots.dtype != torch.int64 or tuple(slots.shape) != (T,):
        _fail(op, f"slots must be int64 [{T}], got {slots.dtype} {tuple(slots.shape)}")
    return slots.contiguous()


# ---- norm and rotation --------------------------------------------------------------------------
def _rope_args(op, q, k, q_weight, k_weight, cos_sin, positions, axis, eps, plus_one, adjacent):
    """(arguments of the C call up to the axes, tensors that they point into)."""
    q, k = _heads(op, "q", q), _heads(op, "k", k)
    T, d = q.shape[0], q.shape[2]
    if k.shape[0] != T or k.shape[2] != d:
        _fail(op, f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    flags = (_native.PLUS_ONE if plus_one else 0) | (_native.ADJACENT if adjacent else 0)
    weights = []
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            if w.dtype != torch.bfloat16 or tuple(w.shape) != (d,):
                _fail(op, f"{name} must be bf16 [{d}], got {w.dtype} {tuple(w.shape)}")
            if w.stride(0) != 1 or w.data_ptr() % 16:
                w = w.clone(memory_format=torch.contiguous_format)
        weights.append(w)
    if cos_sin is None:
        rot, rows, pos_stride, axes = 0, 0, 0, 1
        positions = axis = None
    else:
        if cos_sin.dtype not in (torch.float32, torch.bfloat16) or cos_sin.dim() != 2:
            _fail(op, f"cos_sin must be fp32 or bf16 [positions, rotated channels], got "
                      f"{cos_sin.dtype} {tuple(cos_sin.shape)}")
        rows, rot = cos_sin.shape
        if rot == 0 or rot > d or rot % 16:
            _fail(op, f"{rot} rotated channels: need a multiple of 16 up to the head size {d}")
        cos_sin = cos_sin.contiguous()
        if positions is None or positions.dtype not in (torch.int64, torch.int32) \
                or positions.dim() not in (1, 2) or positions.shape[-1] != T \
                or positions.shape[0] == 0 and positions.dim() == 2:
            _fail(op, f"positions must be int64 or int32 [{T}] or [axes, {T}], got "
                      f"{None if positions is None else (positions.dtype, tuple(positions.shape))}")
        axes = positions.shape[0] if positions.dim() == 2 else 1
        if axes > 1 and axis is None:
            _fail(op, f"positions on {axes} axes need the axis of each pair (rotary_axes)")
        if axis is not None:
            if axis.dtype != torch.int32 or tuple(axis.shape) != (rot // 2,):
                _fail(op, f"axis must be int32 [{rot // 2}], got {axis.dtype} {tuple(axis.shape)}")
            axis = axis.contiguous()
        if positions.stride(-1) != 1 or (axes > 1 and positions.stride(0) < T):
            positions = positions.contiguous()
        pos_stride = positions.stride(0) if axes > 1 else T
        if cos_sin.dtype == torch.bfloat16:
            flags |= _native.TABLE_BF16
        if positions.dtype == torch.int32:
            flags |= _native.POS_I32
    keep = (q, k, *weights, cos_sin, positions, axis)
    tail = (_ptr(weights[0]), _ptr(weights[1]), _ptr(cos_sin), rows, rot, _ptr(positions),
            pos_stride, axes, _ptr(axis))
    return q, k, tail, flags, keep


def _qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor],
                  k_weight: Optional[torch.Tensor], cos_sin: Optional[torch.Tensor],
                  positions: Optional[torch.Tensor], axis: Optional[torch.Tensor], eps: float,
                  plus_one: bool, adjacent: bool) -> tuple[torch.Tensor, torch.Tensor]:
    op = "qk_norm_rope"
    dev = _same_device(op, q, k, q_weight, k_weight, cos_sin, positions, axis)
    with _on(dev):
        q, k, tail, flags, keep = _rope_args(op, q, k, q_weight, k_weight, cos_sin, positions, axis,
                                             eps, plus_one, adjacent)
        T, Hq, d = q.shape
        Hkv = k.shape[1]
        qo = torch.empty((T, Hq, d), dtype=torch.bfloat16, device=dev)
        ko = torch.empty((T, Hkv, d), dtype=torch.bfloat16, device=dev)
        _native.check(_native.lib().kv4_qk_norm_rope(
            q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), *tail, qo.data_ptr(),
            ko.data_ptr(), T, Hq, Hkv, d, eps, flags, _rmx._stream()))
        del keep                        # stream-ordered: reused only after this launch
    return qo, ko


def _qk_norm_rope_fake(q, k, q_weight, k_weight, cos_sin, positions, axis, eps, plus_one, adjacent):
    return (torch.empty(q.shape, dtype=torch.bfloat16, device=q.device),
            torch.empty(k.shape, dtype=torch.bfloat16, device=k.device))


qk_norm_rope_op = torch.library.custom_op("radiance::qk_norm_rope", _qk_norm_rope, mutates_args=())
qk_norm_rope_op.register_fake(_qk_norm_rope_fake)
_call_qk_norm_rope = _rmx.inference_op(qk_norm_rope_op, _qk_norm_rope, _qk_norm_rope_fake)


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
    op = "qk_norm_rope_append"
    dev = _same_device(op, q, k, v, q_weight, k_weight, cos_sin, positions, cache, slots, axis)
    with _on(dev):
        q, k, tail, flags, keep = _rope_args(op, q, k, q_weight, k_weight, cos_sin, positions, axis,
                                             eps, plus_one, adjacent)
        v = _heads(op, "v", v)
        T, Hq, d = q.shape
        Hkv = k.shape[1]
        if tuple(v.shape) != (T, Hkv, d):
            _fail(op, f"v {tuple(v.shape)} does not match k {tuple(k.shape)}")
        page, stride = _cache(op, cache, d, Hkv)
        slots = _slots(op, slots, T)
        qo = torch.empty((T, Hq, d), dtype=torch.bfloat16, device=dev)
        _native.check(_native.lib().kv4_qk_norm_rope_append(
            q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v),
            *tail, qo.data_ptr(), cache.data_ptr(), cache.shape[0], stride, page, slots.data_ptr(),
            T, Hq, Hkv, d, eps, flags, _rmx._stream()))
        del keep                        # stream-ordered: reused only after this launch
    return qo


def _qk_norm_rope_kv4_fake(q, k, v, q_weight, k_weight, cos_sin, positions, cache, slots, axis, eps,
                           plus_one, adjacent):
    return torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)


qk_norm_rope_kv4_op = torch.library.custom_op("radiance::qk_norm_rope_kv4", _qk_norm_rope_kv4,
                                              mutates_args=("cache",))
qk_norm_rope_kv4_op.register_fake(_qk_norm_rope_kv4_fake)
_call_qk_norm_rope_kv4 = _rmx.inference_op(qk_norm_rope_kv4_op, _qk_norm_rope_kv4,
                                           _qk_norm_rope_kv4_fake)


def qk_norm_rope_append(q, k, v, q_weight, k_weight, cos_sin, positions, cache, slots, *, axis=None,
                        eps: float = 1e-6, plus_one: bool = False, adjacent: bool = False):
    """qk_norm_rope, with the keys (rounded from fp32) and the values v [T, kv heads, d] written into
    `cache` at `slots` (int64 [T], distinct; negative ones are skipped, for padding). Returns q."""
    return _call_qk_norm_rope_kv4(q, k, v, q_weight, k_weight, cos_sin, positions, cache, slots, axis,
                                  float(eps), bool(plus_one), bool(adjacent))


# ---- reading back -------------------------------------------------------------------------------
def _kv4_gather(cache: torch.Tensor, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    op = "gather"
    dev = _same_device(op, cache, slots)
    with _on(dev):
        page, stride = _cache(op, cache)
        slots = _slots(op, slots, slots.shape[0] if slots.dim() else 0)
        T, H, d = slots.shape[0], cache.shape[1], cache.shape[3] // 17
        k = torch.empty((T, H, d), dtype=torch.bfloat16, device=dev)
        v = torch.empty((T, H, d), dtype=torch.bfloat16, device=dev)
        _native.check(_native.lib().kv4_gather(cache.data_ptr(), cache.shape[0], stride, page,
                                               slots.data_ptr(), k.data_ptr(), v.data_ptr(), T, H,
                                               d, _rmx._stream()))
    return k, v


def _kv4_gather_fake(cache, slots):
    shape = (slots.shape[0], cache.shape[1], cache.shape[3] // 17)
    return (torch.empty(shape, dtype=torch.bfloat16, device=cache.device),
            torch.empty(shape, dtype=torch.bfloat16, device=cache.device))


kv4_gather_op = torch.library.custom_op("radiance::kv4_gather", _kv4_gather, mutates_args=())
kv4_gather_op.register_fake(_kv4_gather_fake)
_call_kv4_gather = _rmx.inference_op(kv4_gather_op, _kv4_gather, _kv4_gather_fake)


def gather(cache, slots):
    """The keys and values at `slots` (int64 [T]) as bf16 [T, kv heads, d], exactly what the cache
    holds; zeros at a negative slot, NaN at one past the cache."""
    return _call_kv4_gather(cache, slots)


# ---- attention ----------------------------------------------------------------------------------
def _kv4_attention(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor,
                   seq_lens: torch.Tensor, q_starts: torch.Tensor, max_q: int, max_len: int,
                   scale: float, causal: bool, window: int) -> torch.Tensor:
    op = "attention"
    dev = _same_device(op, q, cache, page_table, seq_lens, q_starts)
    with _on(dev):
        q = _heads(op, "q", q)
        total, Hq, d = q.shape
        page, stride = _cache(op, cache, d)
        Hkv = cache.shape[1]
        B = seq_lens.shape[0] if seq_lens.dim() == 1 else -1
        for name, t, shape in (("seq_lens", seq_lens, (B,)), ("q_starts", q_starts, (B + 1,))):
            if t.dtype != torch.int32 or tuple(t.shape) != shape:
                _fail(op, f"{name} must be int32 {list(shape)}, got {t.dtype} {tuple(t.shape)}")
        if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B:
            _fail(op, f"page_table must be int32 [{B}, pages of a sequence], got "
                      f"{page_table.dtype} {tuple(page_table.shape)}")
        seq_lens, q_starts = seq_lens.contiguous(), q_starts.contiguous()
        if page_table.stride(1) != 1 or page_table.stride(0) < 0:
            page_table = page_table.contiguous()
        out = torch.empty((total, Hq, d), dtype=torch.bfloat16, device=dev)
        if total == 0 or B == 0:
            return out
        need = _native.attention_workspace(total, B, max_q, max_len, Hq, Hkv, d, window)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _native.check(_native.lib().kv4_attention(
            q.data_ptr(), *_strides(q), cache.data_ptr(), cache.shape[0], stride, page,
            page_table.data_ptr(), page_table.stride(0) if B > 1 else 0, page_table.shape[1],
            seq_lens.data_ptr(), q_starts.data_ptr(), out.data_ptr(), _ptr(ws), need, total, B, max_q,
            max_len, Hq, Hkv, d, scale, window, _native.CAUSAL if causal else 0, _rmx._stream()))
        del ws                          # stream-ordered: reused only after this launch
    return out


def _kv4_attention_fake(q, cache, page_table, seq_lens, q_starts, max_q, max_len, scale, causal,
                        window):
    return torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)


kv4_attention_op = torch.library.custom_op("radiance::kv4_attention", _kv4_attention,
                                           mutates_args=())
kv4_attention_op.register_fake(_kv4_attention_fake)
_call_kv4_attention = _rmx.inference_op(kv4_attention_op, _kv4_attention, _kv4_attention_fake)


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
    op = "move_pages"
    dev = _same_device(op, cache, page_table)
    layers = cache.shape[0] if cache.dim() == 5 else 1
    one = cache[0] if cache.dim() == 5 and layers else cache
    if layers == 0:
        return
    _, stride = _cache(op, one)
    if pairs.device.type != "cpu" or pairs.dtype != torch.int32 or pairs.dim() != 2 \
            or pairs.shape[1] != 2:
        _fail(op, f"pairs must be int32 [n, 2] (from, to) on the host, got {pairs.dtype} "
                  f"{tuple(pairs.shape)} on {pairs.device}")
    pairs = pairs.contiguous()
    rows = cols = table_stride = 0
    if page_table is not None:
        if page_table.dtype != torch.int32 or page_table.dim() != 2 \
                or (page_table.numel() and page_table.stride(1) != 1 and page_table.shape[1] > 1):
            _fail(op, f"page_table must be int32 [sequences, pages] with contiguous rows, got "
                      f"{page_table.dtype} {tuple(page_table.shape)}")
        rows, cols = page_table.shape
        table_stride = page_table.stride(0) if rows > 1 else cols
    with _on(dev):
        _native.check(_native.lib().kv4_move_pages(
            cache.data_ptr(), layers, cache.stride(0) if layers > 1 else 0, one.shape[0], stride,
            one.shape[1] * one.shape[2] * one.shape[3], pairs.data_ptr(), pairs.shape[0],
            _ptr(page_table) if rows * cols else 0, rows, cols, table_stride, _rmx._stream()))


def _kv4_move_pages_fake(cache, pairs, page_table):
    return None


kv4_move_pages_op = torch.library.custom_op("radiance::kv4_move_pages", _kv4_move_pages,
                                            mutates_args=("cache", "page_table"))
kv4_move_pages_op.register_fake(_kv4_move_pages_fake)
_call_kv4_move_pages = _rmx.inference_op(kv4_move_pages_op, _kv4_move_pages, _kv4_move_pages_fake)


def move_pages(cache, pairs, page_table=None) -> None:
    """Copies page pairs[i, 0] to page pairs[i, 1] (int32 [n, 2] on the host, read before the call
    returns) in a layer's cache or in all layers of one, and replaces the first by the second in
    page_table (int32 [sequences, pages], contiguous rows) where one is given. One launch per 448
    pairs. Refused: a page both read and written, a page written twice and, with a table, a page read
    twice."""
    _call_kv4_move_pages(cache, pairs, page_table)
