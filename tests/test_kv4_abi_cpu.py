"""libkv4_attn.so on the CPU: it loads, exports what include/kv4_attn.h declares, and refuses bad
arguments before touching a GPU (no compute call is made here)."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as KO
from vllm_sly_radiance_amd import _native_kv4 as N
from vllm_sly_radiance_amd import radiance_kv4 as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20                     # an aligned address that is never read


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(N.LIB_PATH):
        pytest.fail(f"{N.LIB_PATH} missing: run __graft_entry__.build() first")
    return N.load_cdll()


def test_header_binding_and_exports_agree(lib):
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "kv4_attn.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"^\s*(?:const\s+)?\w+\*?\s+\*?(kv4_\w+)\s*\(", src, flags=re.M)))
    assert declared == sorted(N.SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", N.LIB_PATH], capture_output=True, text=True,
                         check=True).stdout
    exported = {ln.split()[-1] for ln in out.splitlines() if " T " in ln}
    assert not [f for f in declared if f not in exported]
    assert not [s for s in exported if not s.startswith(("kv4_", "_"))]
    assert lib.kv4_abi_version() == N.ABI_VERSION


def test_page_bytes(lib):
    assert N.page_bytes(8, 16, 128) == 8 * 17 * 128
    assert N.page_bytes(2, 256, 64) == 2 * 16 * 17 * 64
    for heads, page, d, msg in ((0, 16, 128, b"heads"), (8, 24, 128, b"page of 24"),
                                (8, 16, 96, b"head size 96")):
        n = ctypes.c_size_t()
        assert lib.kv4_page_bytes(heads, page, d, ctypes.byref(n)) == N_EINVAL
        assert msg in lib.kv4_last_error()


N_EINVAL = 1


def rope(lib, **kw):
    a = dict(q=P, qts=1024, qhs=128, k=P, kts=1024, khs=128, qw=P, kw=P, table=P, rows=10, rot=128,
             pos=P, ps=4, axes=1, axis=None, qo=P, ko=P, T=4, Hq=4, Hkv=2, d=128, eps=1e-6, flags=0)
    a.update(kw)
    return lib.kv4_qk_norm_rope(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(T=-1), b"T=-1"), (dict(Hq=0), b"heads"), (dict(Hkv=-3), b"heads"), (dict(d=96), b"head size"),
    (dict(rot=24), b"multiple of 16"), (dict(rot=144), b"multiple of 16"), (dict(rot=-16), b"rotated"),
    (dict(axes=0), b"axes"), (dict(axes=2), b"axis of each pair"), (dict(flags=64), b"flags"),
    (dict(q=None), b"null q"), (dict(k=P + 8), b"aligned"), (dict(qts=4), b"strides"),
    (dict(khs=-128), b"strides"), (dict(qw=P + 2), b"weights"), (dict(table=None), b"null table"),
    (dict(pos=None), b"null table or positions"), (dict(pos=P + 4), b"misaligned"),
    (dict(axes=2, axis=P, ps=3), b"position rows"), (dict(qo=None), b"output"), (dict(ko=P + 4), b"output"),
    (dict(rows=-1), b"table rows")])
def test_rope_refuses(lib, kw, msg):
    assert rope(lib, **kw) == N_EINVAL and msg in lib.kv4_last_error()


def test_nothing_to_do_needs_no_gpu(lib):
    assert rope(lib, T=0, q=None, k=None, qo=None, ko=None) == 0
    assert lib.kv4_gather(None, 0, 17 * 128, 16, None, None, None, 0, 1, 128, None) == 0
    assert lib.kv4_attention(None, 0, 0, None, 0, 17 * 128, 16, None, 0, 0, None, None, None, None, 0, 0,
                             3, 1, 10, 2, 1, 128, 1.0, 0, 0, None) == 0
    assert lib.kv4_move_pages(P, 2, 1 << 20, 4, 17 * 64, 17 * 64, None, 0, None, 0, 0, 0, None) == 0


def append(lib, **kw):
    a = dict(q=P, qts=1024, qhs=128, k=P, kts=1024, khs=128, v=P, vts=1024, vhs=128, qw=None, kw=None,
             table=None, rows=0, rot=0, pos=None, ps=0, axes=1, axis=None, qo=P, cache=P, pages=5,
             stride=2 * 17 * 128, page=16, slots=P, T=4, Hq=4, Hkv=2, d=128, eps=1e-6, flags=0)
    a.update(kw)
    return lib.kv4_qk_norm_rope_append(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(page=8), b"page of 8"), (dict(page=48), b"page of 48"), (dict(pages=-1), b"pages"),
    (dict(stride=17 * 128), b"page stride"), (dict(stride=2 * 17 * 128 + 8), b"page stride"),
    (dict(cache=None), b"null cache"), (dict(cache=P + 8), b"16-byte"), (dict(slots=None), b"slots"),
    (dict(slots=P + 4), b"slots"), (dict(v=None), b"null v"), (dict(vhs=12), b"strides"),
    (dict(qo=None), b"output")])
def test_append_refuses(lib, kw, msg):
    assert append(lib, **kw) == N_EINVAL and msg in lib.kv4_last_error()


def attention(lib, **kw):
    a = dict(q=P, qts=512, qhs=128, cache=P, pages=9, stride=2 * 17 * 128, page=16, table=P, ts=4, cols=4,
             lens=P, starts=P, out=P, ws=None, wsb=0, total=3, batch=2, max_q=2, max_len=60, Hq=4, Hkv=2,
             d=128, scale=0.1, window=0, flags=N.CAUSAL)
    a.update(kw)
    return lib.kv4_attention(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(Hq=5), b"5 query heads over 2"), (dict(Hkv=0), b"heads"), (dict(d=80), b"head size"),
    (dict(batch=-1), b"batch=-1"), (dict(max_q=-1), b"max_q=-1"), (dict(max_len=-5), b"max_len=-5"),
    (dict(window=-1), b"window=-1"), (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"),
    (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"),
    (dict(flags=1), b"flags"), (dict(total=-1), b"total=-1"), (dict(cols=-1), b"table_cols=-1"),
    (dict(q=P + 2), b"aligned"), (dict(qhs=100), b"strides"), (dict(lens=None), b"null pointer"),
    (dict(starts=P + 2), b"misaligned"), (dict(out=P + 8), b"misaligned"), (dict(table=None), b"null"),
    (dict(page=100), b"page of 100"), (dict(stride=100), b"page stride"),
    (dict(max_len=100000, cols=6250), b"workspace"),
    (dict(max_len=100000, cols=6250, ws=P + 4, wsb=1 << 40), b"workspace"),
    (dict(batch=1 << 20, max_q=1 << 20), b"too many rows")])
def test_attention_refuses(lib, kw, msg):
    assert attention(lib, **kw) == N_EINVAL and msg in lib.kv4_last_error()


def move(lib, pairs, pages=10, layers=2, layer=1 << 20, stride=17 * 64, size=17 * 64, cache=P, tables=None,
         rows=0, cols=0, ts=0):
    p = np.asarray(pairs, np.int32).reshape(-1, 2)
    return lib.kv4_move_pages(cache, layers, layer, pages, stride, size, p.ctypes.data, len(p), tables,
                              rows, cols, ts, None)


@pytest.mark.parametrize("pairs,kw,msg", [
    ([[1, 10]], {}, b"outside the 10 pages"), ([[-1, 2]], {}, b"outside"),
    ([[1, 2], [3, 2]], {}, b"page 2 is written twice"), ([[1, 2], [2, 3]], {}, b"page 2 is both"),
    ([[4, 4]], {}, b"page 4 is both"), ([[1, 2], [1, 3]], dict(tables=P, rows=1, cols=4, ts=4), b"two places"),
    ([[1, 2]], dict(stride=16), b"page stride"), ([[1, 2]], dict(size=17 * 64 + 8), b"multiples of 16"),
    ([[1, 2]], dict(cache=None), b"null"), ([[1, 2]], dict(layers=-1), b"layers=-1"),
    ([[1, 2]], dict(tables=P, rows=2, cols=5, ts=4), b"row stride"),
    ([[i, 50 + i] for i in range(11)], {}, b"11 pairs over 10 pages")])
def test_move_refuses(lib, pairs, kw, msg):
    assert move(lib, pairs, **kw) == N_EINVAL and msg in lib.kv4_last_error()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_oracle_layout_is_a_permutation_and_reads_back(d):
    at = np.concatenate([np.concatenate(KO.places(t, d)) for t in range(16)])
    assert np.array_equal(np.sort(at), np.arange(17 * d))
    rng = np.random.default_rng(d)
    cache = np.zeros((3, 2, 2, 17 * d), np.uint8)
    slots = rng.permutation(96)[:50]
    k = rng.standard_normal((50, 2, d)).astype(np.float32) * 4
    v = rng.standard_normal((50, 2, d)).astype(np.float32) / 64
    KO.write(cache, slots, k, v)
    for x, y in zip((k, v), KO.read(cache, slots)):
        top = np.abs(x.reshape(50, 2, -1, 32)).max(-1)
        # a code is off by at most half its step: 1 of the scale at the top, and top > 3.5 of it
        assert (np.abs(x - y).reshape(50, 2, -1, 32).max(-1) <= top / 3.5).all()
        assert np.linalg.norm(x - y) / np.linalg.norm(x) < 0.2


def test_oracle_rounding_known_answers():
    x = np.zeros((1, 32), np.float32)
    x[0, :9] = [7.0, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -6.5]
    c, e = KO.quantize(x)
    assert e[0, 0] == 127 and c[0, :9].tolist() == [7, 6, 6, 4, 4, 2, 2, 0, 15]
    x[0, 0] = np.nextafter(np.float32(7), np.float32(8))
    assert KO.quantize(x)[1][0, 0] == 128
    x[0, 0] = np.inf
    assert KO.quantize(x)[1][0, 0] == 255 and np.isnan(KO.dequantize(*KO.quantize(x))).all()
    x[:] = 3.4e38
    assert KO.quantize(x)[1][0, 0] == 252
    x[:] = 0
    assert KO.quantize(x)[1][0, 0] == 1


def test_rotary_axes():
    ax = lambda *a, **k: K.rotary_axes(*a, device="cpu", **k).tolist()  # noqa: E731
    assert ax([2, 3, 1]) == [0, 0, 1, 1, 1, 2]
    assert ax([4, 2, 2], interleaved=True) == [0, 1, 2, 0, 1, 2, 0, 0]
    for bad in ([], [0, 0], [3, -1]):
        with pytest.raises(RuntimeError, match="sections"):
            ax(bad)
    with pytest.raises(RuntimeError, match="interleaved"):
        ax([1, 5], interleaved=True)


def test_python_refusals_need_no_gpu():
    t = torch.zeros((2, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="on the GPU"):
        K.qk_norm_rope(t, t, None, None, None, None)
    with pytest.raises(RuntimeError, match="head size"):
        K.new_cache(2, 2, 16, 96, device="cpu")
    with pytest.raises(RuntimeError, match="page"):
        K.new_cache(2, 2, 24, 128, device="cpu")
    c = K.new_cache(3, 2, 32, 64, device="cpu", layers=4)
    assert tuple(c.shape) == (4, 3, 2, 2, 17 * 64) and not c.any()


def test_fakes_give_the_outputs_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q = torch.empty((5, 4, 128), dtype=torch.bfloat16, device="cuda")
        k = torch.empty((5, 2, 128), dtype=torch.bfloat16, device="cuda")
        cache = torch.empty((7, 2, 1, 17 * 128), dtype=torch.uint8, device="cuda")
        i = torch.empty(5, dtype=torch.int64, device="cuda")
        n = torch.empty(3, dtype=torch.int32, device="cuda")
        table = torch.empty((3, 4), dtype=torch.int32, device="cuda")
        a, b = K.qk_norm_rope(q, k, None, None, None, None)
        assert a.shape == q.shape and b.shape == k.shape
        assert K.qk_norm_rope_append(q, k, k, None, None, None, None, cache, i).shape == q.shape
        a, b = K.gather(cache, i)
        assert a.shape == b.shape == (5, 2, 128) and a.dtype == torch.bfloat16
        o = K.attention(q, cache, table, n, torch.empty(4, dtype=torch.int32, device="cuda"), 5, 60)
        assert o.shape == q.shape and o.dtype == torch.bfloat16


def workspace(lib, *sizes):
    n = ctypes.c_size_t()
    assert lib.kv4_attention_workspace(*sizes, ctypes.byref(n)) == 0
    return n.value


def test_what_serves_a_call(lib):
    """(total, batch, max_q, max_len, q heads, kv heads, d, window) and the workspace: few rows over a long
    context are shared out over 512 workgroups, two partial results each; many rows (more than 128 a kv
    head, 64 at head size 256, and 200 times half that in all) take a workgroup for each 256 (128), the
    last round's in parts; sequences of few rows beside them, both."""
    few = lambda runs, rows, d: runs * (2 * rows * (d + 2) * 4 + 16)  # noqa: E731
    many = lambda parts, rows, d: parts * rows * (d + 2) * 4 + 4096  # noqa: E731
    assert workspace(lib, 1, 1, 1, 1024, 32, 8, 128, 0) == 0
    assert workspace(lib, 1, 1, 1, 1025, 32, 8, 128, 0) == few(8 * 9, 16, 128)
    assert workspace(lib, 16, 16, 1, 2048, 32, 8, 128, 0) == 0            # 128 units of 8 steps
    assert workspace(lib, 15, 15, 1, 2048, 32, 8, 128, 0) == few(1024, 16, 128)
    assert workspace(lib, 99, 99, 1, 4097, 32, 8, 128, 0) == few(1024, 16, 128)
    assert workspace(lib, 99, 99, 1, 9999, 32, 8, 128, 1000) == 0         # what a window leaves
    assert workspace(lib, 0, 1, 0, 4096, 32, 8, 128, 0) == 0
    assert workspace(lib, 399, 1, 399, 4096, 32, 8, 128, 0) == few(512, 64, 128)
    assert workspace(lib, 400, 1, 400, 4096, 32, 8, 128, 0) == many(56 * 4, 256, 128)
    assert workspace(lib, 400, 1, 400, 400, 32, 8, 128, 0) == 0
    assert workspace(lib, 64 * 32, 64, 32, 4096, 32, 8, 128, 0) == few(512, 64, 128)
    assert workspace(lib, 64 * 33, 64, 33, 4096, 32, 8, 128, 0) == 0      # 512 units, two rounds
    assert workspace(lib, 400, 1, 400, 4096, 16, 2, 256, 0) == many(50 * 5, 128, 256)
    assert workspace(lib, 400, 1, 400, 4096, 64, 64, 64, 0) == many(128 * 2, 256, 64)
    # beside chunks: rows of one query of the group's heads, if they fit attn_rows' 64
    assert workspace(lib, 401, 2, 400, 4096, 65, 1, 128, 0) == many(512, 256, 128)
    assert workspace(lib, 401, 2, 400, 4096, 64, 1, 128, 0) == many(512, 256, 128) + few(64, 64, 128)


def test_binding_refuses():
    """What is no tensor, no number or too many is a Python exception, not a crash."""
    ops = N.ops()
    t = torch.zeros((2, 2, 128), dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    for call, error, what in (
            (lambda: ops.gather(t), RuntimeError, "gather: 1 arguments in place of 2"),
            (lambda: ops.gather(t, 3), RuntimeError, "argument 1 must be a tensor"),
            (lambda: ops.gather(None, t), RuntimeError, "argument 0 must be a tensor"),
            (lambda: ops.gather(t, i), RuntimeError, "on the GPU, got cpu"),
            (lambda: ops.move_pages(t, i, None), RuntimeError, "on the GPU"),
            (lambda: ops.attention(t, t, i, i, i, 2 ** 40, 1, 1.0, True, 0), RuntimeError,
             "max_q=1099511627776 is out of range"),
            (lambda: ops.attention(t, t, i, i, i, 1, -2 ** 70, 1.0, True, 0), OverflowError, ""),
            (lambda: ops.attention(t, t, i, i, i, "1", 1, 1.0, True, 0), TypeError, ""),
            (lambda: ops.attention(t, t, i, i, i, 1, 1, None, True, 0), TypeError, ""),
            (lambda: ops.qk_norm_rope(t, t, None, None, None, None, None, 1e-6, 0, 0), RuntimeError,
             "on the GPU")):
        with pytest.raises(error, match=what or None):
            call()
