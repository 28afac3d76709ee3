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

import functools
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
# The calls below are a few microseconds of GPU work where a batch is small, so the host's share is kept
# small as well: shapes, strides and pointers are read once, and where nothing watches ops by name
# the body is called without the dispatcher (one token through qk_norm_rope, 5 us on the GPU: 18.9
# us a call with the dispatcher and separate helpers, 13.3 now, 2.7 of them the launch).
def _heads(op: str, name: str, x: torch.Tensor):
    """bf16 [T, heads, d] whose heads are 16-byte aligned runs, other layouts copied: (x, T, heads, d,
    its address, token and head strides; those of an axis of one, which may be anything, as 0)."""
    if x.dtype is not torch.bfloat16 or x.dim() != 3:
        _fail(op, f"{name} must be bf16 [tokens, heads, head size], got {x.dtype} {tuple(x.shape)}")
    T, H, d = x.shape
    if d not in HEAD_SIZES:
        _fail(op, f"head size {d} of {name} is none of {HEAD_SIZES}")
    st, sh, sc = x.stride()
    at = x.data_ptr()
    if T <= 1:
        st = 0
    if H <= 1:
        sh = 0
    if (sc != 1 or (st | sh) & 7 or at & 15) and T:
        x = x.clone(memory_format=torch.contiguous_format)
        return _heads(op, name, x)
    return x, T, H, d, at, st, sh


def _cache(op: str, cache: torch.Tensor, d: Optional[int] = None, heads: Optional[int] = None):
    """(pages, kv heads, page size, head size, page stride) of a layer's cache."""
    if cache.dtype is not torch.uint8 or cache.dim() != 4 or cache.shape[3] % 17 \
            or cache.shape[3] // 17 not in HEAD_SIZES or cache.shape[2] * GROUP not in PAGE_SIZES:
        _fail(op, f"cache must be uint8 [pages, kv heads, page / 16, 17 * head size], got "
                  f"{cache.dtype} {tuple(cache.shape)}")
    pages, H, n, b = cache.shape
    sp, sh, sn, sb = cache.stride()
    if (sb != 1 or (n > 1 and sn != b) or (H > 1 and sh != n * b) or cache.data_ptr() & 15) \
            and cache.numel():
        _fail(op, "a page of the cache must be contiguous and 16-byte aligned")
    if d is not None and b != 17 * d:
        _fail(op, f"cache of head size {b // 17} against {d}")
    if heads is not None and H != heads:
        _fail(op, f"cache of {H} kv heads against {heads}")
    return pages, H, n * GROUP, b // 17, sp if pages > 1 else H * n * b


def _same_device(op: str, *tensors):
    dev = tensors[0].device
    if dev.type != "cuda":
        _fail(op, f"tensors must be on the GPU, got {dev}")
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            _fail(op, f"tensors on {dev} and {t.device}")
    return dev


def _entry(op, body):
    """The body, called on the tensors' device; through `op`, whose name a compiler, a tracer or a mode
    then sees and whose backward raises, where one watches or a gradient may be asked for."""
    ns, name = op._qualname.split("::")
    space = getattr(torch.ops, ns)

    def call(*args):
        if _rmx._watched() or type(args[0]) is not torch.Tensor \
                or (torch.is_grad_enabled() and _rmx._asks_gradient(args)):
            return getattr(space, name)(*args)
        return body(*args)
    return call


def _on_device(body):
    """body with the device of its first argument, a GPU's tensor, as the current one."""
    @functools.wraps(body)
    def run(first, *args):
        if first.is_cuda and first.get_device() != torch._C._cuda_getDevice():
            with torch.cuda.device(first.device):
                return body(first, *args)
        return body(first, *args)
    return run


def _stream(dev) -> int:
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _slots(op: str, slots: torch.Tensor, T: int) -> torch.Tensor:
    if slots.dtype is not torch.int64 or slots.dim() != 1 or slots.shape[0] != T:
        _fail(op, f"slots must be int64 [{T}], got {slots.dtype} {tuple(slots.shape)}")
    return slots.contiguous()


# ---- norm and rotation --------------------------------------------------------------------------
def _rope_args(op, T, d, q_weight, k_weight, cos_sin, positions, axis, plus_one, adjacent):
    """(the C call's arguments from the weights to the axes, flags, tensors that they point into)."""
    flags = (_native.PLUS_ONE if plus_one else 0) | (_native.ADJACENT if adjacent else 0)
    weights, at = [], []
    for w in (q_weight, k_weight):
        p = 0
        if w is not None:
            if w.dtype is not torch.bfloat16 or w.dim() != 1 or w.shape[0] != d:
                _fail(op, f"{'k_weight' if weights else 'q_weight'} must be bf16 [{d}], got {w.dtype} "
                          f"{tuple(w.shape)}")
            p = w.data_ptr()
            if p & 15 or w.stride(0) != 1:
                w = w.clone(memory_format=torch.contiguous_format)
                p = w.data_ptr()
        weights.append(w)
        at.append(p)
    if cos_sin is None:
        return (*at, 0, 0, 0, 0, 0, 1, 0), flags, weights
    fp32 = cos_sin.dtype is torch.float32
    if not (fp32 or cos_sin.dtype is torch.bfloat16) or cos_sin.dim() != 2:
        _fail(op, f"cos_sin must be fp32 or bf16 [positions, rotated channels], got "
                  f"{cos_sin.dtype} {tuple(cos_sin.shape)}")
    rows, rot = cos_sin.shape
    if rot == 0 or rot > d or rot % 16:
        _fail(op, f"{rot} rotated channels: need a multiple of 16 up to the head size {d}")
    cos_sin = cos_sin.contiguous()
    dims = 0 if positions is None else positions.dim()
    i32 = dims and positions.dtype is torch.int32
    if dims not in (1, 2) or not (i32 or positions.dtype is torch.int64) \
            or positions.shape[-1] != T or positions.shape[0] == 0 and dims == 2:
        _fail(op, f"positions must be int64 or int32 [{T}] or [axes, {T}], got "
                  f"{None if positions is None else (positions.dtype, tuple(positions.shape))}")
    axes = positions.shape[0] if dims == 2 else 1
    if axes > 1 and axis is None:
        _fail(op, f"positions on {axes} axes need the axis of each pair (rotary_axes)")
    if axis is not None:
        if axis.dtype is not torch.int32 or tuple(axis.shape) != (rot // 2,):
            _fail(op, f"axis must be int32 [{rot // 2}], got {axis.dtype} {tuple(axis.shape)}")
        axis = axis.contiguous()
    if positions.stride(-1) != 1 or (axes > 1 and positions.stride(0) < T):
        positions = positions.contiguous()
    flags |= (0 if fp32 else _native.TABLE_BF16) | (_native.POS_I32 if i32 else 0)
    return ((*at, cos_sin.data_ptr(), rows, rot, positions.data_ptr(),
             positions.stride(0) if axes > 1 else T, axes, _ptr(axis)), flags,
            (weights, cos_sin, positions, axis))


def _same_tokens(op, T, d, name, x, xT, xd):
    if xT != T or xd != d:
        _fail(op, f"{name} {tuple(x.shape)} does not match q [{T}, ..., {d}]")


@_on_device
def _qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor],
                  k_weight: Optional[torch.Tensor], cos_sin: Optional[torch.Tensor],
                  positions: Optional[torch.Tensor], axis: Optional[torch.Tensor], eps: float,
                  plus_one: bool, adjacent: bool) -> tuple[torch.Tensor, torch.Tensor]:
    op = "qk_norm_rope"
    dev = _same_device(op, q, k, q_weight, k_weight, cos_sin, positions, axis)
    q, T, Hq, d, qp, qt, qh = _heads(op, "q", q)
    k, kT, Hkv, kd, kp, kt, kh = _heads(op, "k", k)
    _same_tokens(op, T, d, "k", k, kT, kd)
    tail, flags, keep = _rope_args(op, T, d, q_weight, k_weight, cos_sin, positions, axis, plus_one,
                                   adjacent)
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    ko = torch.empty_like(k, memory_format=torch.contiguous_format)
    # (q, k and keep may be copies: stream-ordered, reused only after this launch)
    _native.check(_native.lib().kv4_qk_norm_rope(
        qp, qt, qh, kp, kt, kh, *tail, qo.data_ptr(), ko.data_ptr(), T, Hq, Hkv, d, eps, flags,
        _stream(dev)))
    return qo, ko


def _qk_norm_rope_fake(q, k, q_weight, k_weight, cos_sin, positions, axis, eps, plus_one, adjacent):
    return (torch.empty(q.shape, dtype=torch.bfloat16, device=q.device),
            torch.empty(k.shape, dtype=torch.bfloat16, device=k.device))


qk_norm_rope_op = torch.library.custom_op("radiance::qk_norm_rope", _qk_norm_rope, mutates_args=())
qk_norm_rope_op.register_fake(_qk_norm_rope_fake)
_call_qk_norm_rope = _entry(qk_norm_rope_op, _qk_norm_rope)


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


@_on_device
def _qk_norm_rope_kv4(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                      cos_sin: Optional[torch.Tensor], positions: Optional[torch.Tensor],
                      cache: torch.Tensor, slots: torch.Tensor, axis: Optional[torch.Tensor],
                      eps: float, plus_one: bool, adjacent: bool) -> torch.Tensor:
    op = "qk_norm_rope_append"
    dev = _same_device(op, q, k, v, q_weight, k_weight, cos_sin, positions, cache, slots, axis)
    q, T, Hq, d, qp, qt, qh = _heads(op, "q", q)
    k, kT, Hkv, kd, kp, kt, kh = _heads(op, "k", k)
    v, vT, Hv, vd, vp, vt, vh = _heads(op, "v", v)
    _same_tokens(op, T, d, "k", k, kT, kd)
    _same_tokens(op, T, d, "v", v, vT, vd)
    if Hv != Hkv:
        _fail(op, f"v {tuple(v.shape)} does not match k {tuple(k.shape)}")
    tail, flags, keep = _rope_args(op, T, d, q_weight, k_weight, cos_sin, positions, axis, plus_one,
                                   adjacent)
    pages, _, page, _, stride = _cache(op, cache, d, Hkv)
    slots = _slots(op, slots, T)
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    # (the inputs may be copies: stream-ordered, reused only after this launch)
    _native.check(_native.lib().kv4_qk_norm_rope_append(
        qp, qt, qh, kp, kt, kh, vp, vt, vh, *tail, qo.data_ptr(), cache.data_ptr(), pages, stride,
        page, slots.data_ptr(), T, Hq, Hkv, d, eps, flags, _stream(dev)))
    return qo


def _qk_norm_rope_kv4_fake(q, k, v, q_weight, k_weight, cos_sin, positions, cache, slots, axis, eps,
                           plus_one, adjacent):
    return torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)


qk_norm_rope_kv4_op = torch.library.custom_op("radiance::qk_norm_rope_kv4", _qk_norm_rope_kv4,
                                              mutates_args=("cache",))
qk_norm_rope_kv4_op.register_fake(_qk_norm_rope_kv4_fake)
_call_qk_norm_rope_kv4 = _entry(qk_norm_rope_kv4_op, _qk_norm_rope_kv4)


def qk_norm_rope_append(q, k, v, q_weight, k_weight, cos_sin, positions, cache, slots, *, axis=None,
                        eps: float = 1e-6, plus_one: bool = False, adjacent: bool = False):
    """qk_norm_rope, with the keys (rounded from fp32) and the values v [T, kv heads, d] written into
    `cache` at `slots` (int64 [T], distinct; negative ones are skipped, for padding). Returns q."""
    return _call_qk_norm_rope_kv4(q, k, v, q_weight, k_weight, cos_sin, positions, cache, slots, axis,
                                  float(eps), bool(plus_one), bool(adjacent))


# ---- reading back -------------------------------------------------------------------------------
@_on_device
def _kv4_gather(cache: torch.Tensor, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    op = "gather"
    dev = _same_device(op, cache, slots)
    pages, H, page, d, stride = _cache(op, cache)
    slots = _slots(op, slots, slots.shape[0] if slots.dim() else 0)
    T = slots.shape[0]
    k = torch.empty((T, H, d), dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    _native.check(_native.lib().kv4_gather(cache.data_ptr(), pages, stride, page, slots.data_ptr(),
                                           k.data_ptr(), v.data_ptr(), T, H, d, _stream(dev)))
    return k, v


def _kv4_gather_fake(cache, slots):
    shape = (slots.shape[0], cache.shape[1], cache.shape[3] // 17)
    return (torch.empty(shape, dtype=torch.bfloat16, device=cache.device),
            torch.empty(shape, dtype=torch.bfloat16, device=cache.device))


kv4_gather_op = torch.library.custom_op("radiance::kv4_gather", _kv4_gather, mutates_args=())
kv4_gather_op.register_fake(_kv4_gather_fake)
_call_kv4_gather = _entry(kv4_gather_op, _kv4_gather)


def gather(cache, slots):
    """The keys and values at `slots` (int64 [T]) as bf16 [T, kv heads, d], exactly what the cache
    holds; zeros at a negative slot, NaN at one past the cache."""
    return _call_kv4_gather(cache, slots)


# ---- attention ----------------------------------------------------------------------------------
@_on_device
def _kv4_attention(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor,
                   seq_lens: torch.Tensor, q_starts: torch.Tensor, max_q: int, max_len: int,
                   scale: float, causal: bool, window: int) -> torch.Tensor:
    op = "attention"
    dev = _same_device(op, q, cache, page_table, seq_lens, q_starts)
    q, total, Hq, d, qp, qt, qh = _heads(op, "q", q)
    pages, Hkv, page, _, stride = _cache(op, cache, d)
    B = seq_lens.shape[0] if seq_lens.dim() == 1 else -1
    if seq_lens.dtype is not torch.int32 or B < 0:
        _fail(op, f"seq_lens must be int32 [batch], got {seq_lens.dtype} {tuple(seq_lens.shape)}")
    if q_starts.dtype is not torch.int32 or q_starts.dim() != 1 or q_starts.shape[0] != B + 1:
        _fail(op, f"q_starts must be int32 [{B + 1}], got {q_starts.dtype} {tuple(q_starts.shape)}")
    if page_table.dtype is not torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B:
        _fail(op, f"page_table must be int32 [{B}, pages of a sequence], got "
                  f"{page_table.dtype} {tuple(page_table.shape)}")
    seq_lens, q_starts = seq_lens.contiguous(), q_starts.contiguous()
    row, col = page_table.stride()
    if col != 1:
        page_table = page_table.contiguous()
        row = page_table.stride(0)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if total == 0 or B == 0:
        return out
    need = _native.attention_workspace(total, B, max_q, max_len, Hq, Hkv, d, window)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    # (the workspace and inputs that are copies: stream-ordered, reused only after this launch)
    _native.check(_native.lib().kv4_attention(
        qp, qt, qh, cache.data_ptr(), pages, stride, page, page_table.data_ptr(), row if B > 1 else 0,
        page_table.shape[1], seq_lens.data_ptr(), q_starts.data_ptr(), out.data_ptr(), _ptr(ws), need,
        total, B, max_q, max_len, Hq, Hkv, d, scale, window, _native.CAUSAL if causal else 0,
        _stream(dev)))
    return out


def _kv4_attention_fake(q, cache, page_table, seq_lens, q_starts, max_q, max_len, scale, causal,
                        window):
    return torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)


kv4_attention_op = torch.library.custom_op("radiance::kv4_attention", _kv4_attention,
                                           mutates_args=())
kv4_attention_op.register_fake(_kv4_attention_fake)
_call_kv4_attention = _entry(kv4_attention_op, _kv4_attention)


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
@_on_device
def _kv4_move_pages(cache: torch.Tensor, pairs: torch.Tensor,
                    page_table: Optional[torch.Tensor]) -> None:
    op = "move_pages"
    dev = _same_device(op, cache, page_table)
    layers = cache.shape[0] if cache.dim() == 5 else 1
    one = cache[0] if cache.dim() == 5 and layers else cache
    if layers == 0:
        return
    pages, heads, page, d, stride = _cache(op, one)
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
    _native.check(_native.lib().kv4_move_pages(
        cache.data_ptr(), layers, cache.stride(0) if layers > 1 else 0, pages, stride,
        heads * page // GROUP * 17 * d, pairs.data_ptr(), pairs.shape[0],
        _ptr(page_table) if rows * cols else 0, rows, cols, table_stride, _stream(dev)))


def _kv4_move_pages_fake(cache, pairs, page_table):
    return None


kv4_move_pages_op = torch.library.custom_op("radiance::kv4_move_pages", _kv4_move_pages,
                                            mutates_args=("cache", "page_table"))
kv4_move_pages_op.register_fake(_kv4_move_pages_fake)
_call_kv4_move_pages = _entry(kv4_move_pages_op, _kv4_move_pages)


def move_pages(cache, pairs, page_table=None) -> None:
    """Copies page pairs[i, 0] to page pairs[i, 1] (int32 [n, 2] on the host, read before the call
    returns) in a layer's cache or in all layers of one, and replaces the first by the second in
    page_table (int32 [sequences, pages], contiguous rows) where one is given. One launch per 448
    pairs. Refused: a page both read and written, a page written twice and, with a table, a page read
    twice."""
    _call_kv4_move_pages(cache, pairs, page_table)
