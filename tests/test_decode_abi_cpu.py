"""libdecode_ops.so on the CPU: it loads, exports what include/decode_ops.h declares, and refuses bad
arguments before touching a GPU (no compute call is made here)."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from vllm_sly_radiance_amd import _native_decode as N
from vllm_sly_radiance_amd import radiance_gdn as G
from vllm_sly_radiance_amd import radiance_sample as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20                     # an aligned address that is never read
EINVAL = 1


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(N.LIB_PATH):
        pytest.fail(f"{N.LIB_PATH} missing: run __graft_entry__.build() first")
    return N.load_cdll()


def test_header_binding_and_exports_agree(lib):
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "decode_ops.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"^\s*(?:const\s+)?\w+\*?\s+\*?(dec_\w+)\s*\(", src, flags=re.M)))
    assert declared == sorted(N.SIGNATURES)
    for name in declared:
        args = re.search(name + r"\s*\((.*?)\);", src, flags=re.S).group(1)
        count = 0 if args.strip() == "void" else args.count(",") + 1
        assert count == len(N.SIGNATURES[name][1]), name
    out = subprocess.run(["nm", "-D", "--defined-only", N.LIB_PATH], capture_output=True, text=True,
                         check=True).stdout
    exported = {ln.split()[-1] for ln in out.splitlines() if " T " in ln}
    assert not [f for f in declared if f not in exported]
    assert not [s for s in exported if not s.startswith(("dec_", "_"))]
    assert lib.dec_abi_version() == N.ABI_VERSION


def test_header_is_c():
    code = '#include "decode_ops.h"\nint main(void) { return DEC_OK; }\n'
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"),
                    "-x", "c", "-"], input=code, text=True, check=True)


def conv(lib, **kw):
    a = dict(x=P, ts=64, w=P, bias=P, state=P, slots=4, ss=192, starts=P, read=P, write=P, ws=1, wc=0, out=P, T=5,
             B=2, mq=3, C=64, W=4, flags=N.SILU)
    a.update(kw)
    return lib.dec_causal_conv(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(T=-1), b"total=-1"), (dict(B=-1), b"batch=-1"), (dict(mq=-1), b"max_q=-1"), (dict(C=12), b"12 channels"),
    (dict(C=0), b"0 channels"), (dict(C=-8), b"channels"), (dict(W=1), b"width 1"), (dict(W=5), b"width 5"),
    (dict(flags=64), b"flags"), (dict(slots=-1), b"-1 slots"), (dict(slots=1 << 31), b"slots"),
    (dict(ss=184), b"slot stride"), (dict(ss=196), b"slot stride"), (dict(ss=1 << 61), b"slot stride"),
    (dict(wc=-1), b"write slots"), (dict(wc=3, ws=2), b"write slots"), (dict(ws=0), b"write slots"),
    (dict(ws=-1), b"write slots"), (dict(starts=None), b"starts"), (dict(read=None), b"starts or slots"),
    (dict(write=P + 2), b"misaligned starts"), (dict(state=None), b"null state"), (dict(state=P + 8), b"state"),
    (dict(w=None), b"weight"), (dict(w=P + 8), b"weight"), (dict(bias=P + 2), b"bias"), (dict(x=None), b"null x"),
    (dict(x=P + 2), b"aligned"), (dict(ts=68), b"strides"), (dict(ts=-64), b"strides"), (dict(out=None), b"output"),
    (dict(out=P + 8), b"output"), (dict(B=1 << 30), b"too large")])
def test_conv_refuses(lib, kw, msg):
    assert conv(lib, **kw) == EINVAL and msg in lib.dec_last_error()


def delta(lib, **kw):
    a = dict(q=P, qts=256, qhs=128, k=P, kts=256, khs=128, v=P, vts=512, vhs=128, a=P, ats=4, b=P, bts=4, al=P, dt=P,
             state=P, slots=3, ss=4 * 128 * 128, starts=P, read=P, write=P, ws=1, wc=0, out=P, work=P, wb=1 << 40, T=5,
             B=2, mq=3, Hk=2, Hv=4, dk=128, dv=128, scale=0.1, eps=1e-6)
    a.update(kw)
    return lib.dec_gated_delta(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(T=-1), b"total=-1"), (dict(B=-2), b"batch=-2"), (dict(mq=-1), b"max_q"), (dict(wc=-1), b"write_cols=-1"),
    (dict(Hk=0), b"heads"), (dict(Hv=5), b"5 value heads over 2"), (dict(Hv=0), b"heads"), (dict(Hv=8192), b"heads"),
    (dict(dk=96), b"96 and 128"), (dict(dv=256), b"none of 64, 128"), (dict(dk=0), b"none of"),
    (dict(slots=-1), b"slots"), (dict(ss=4 * 128 * 127), b"slot stride"), (dict(ss=4 * 128 * 128 + 2), b"slot stride"),
    (dict(ws=0), b"write slots"), (dict(scale=float("nan")), b"scale"), (dict(eps=-1.0), b"eps"),
    (dict(eps=float("nan")), b"eps"), (dict(starts=None), b"starts"), (dict(read=P + 1), b"misaligned"),
    (dict(write=None), b"null"), (dict(state=None), b"state"), (dict(state=P + 4), b"state"), (dict(al=None), b"a_log"),
    (dict(dt=P + 2), b"dt_bias"), (dict(q=None), b"null q"), (dict(k=P + 8), b"k needs"), (dict(vts=516), b"v needs"),
    (dict(qhs=-128), b"strides"), (dict(a=None), b"null or misaligned a"), (dict(b=P + 1), b"misaligned a or b"),
    (dict(ats=-1), b"strides -1"), (dict(out=None), b"output"), (dict(B=1 << 28), b"too large")])
def test_delta_refuses(lib, kw, msg):
    assert delta(lib, **kw) == EINVAL and msg in lib.dec_last_error()


def test_delta_wants_its_workspace(lib):
    n = N.gated_delta_workspace(5000, 2, 4000, 0, 2, 4, 128, 128)
    assert n >= 0 and n % 16 == 0
    for T, mq in ((5000, 4000), (1 << 22, 1 << 21)):
        need = N.gated_delta_workspace(T, 2, mq, 0, 2, 4, 128, 128)
        if need:
            for kw in (dict(wb=need - 1), dict(work=None), dict(work=P + 8)):
                assert delta(lib, T=T, mq=mq, **kw) == EINVAL and b"workspace" in lib.dec_last_error()
    assert N.gated_delta_workspace(64, 64, 1, 0, 2, 4, 128, 128) == 0     # decoding takes none
    with pytest.raises(RuntimeError, match="none of 64, 128"):
        N.gated_delta_workspace(64, 64, 1, 0, 2, 4, 128, 32)
    assert lib.dec_gated_delta_workspace(64, 64, 1, 0, 2, 4, 128, 128, None) == EINVAL


def sample(lib, **kw):
    a = dict(x=P, stride=100, u=P, t=P, ta=1.0, k=P, ka=0, p=P, pa=1.0, mp=P, ma=0.0, tokens=P, lp=P, work=P,
             wb=1 << 40, rows=3, V=100, flags=N.LOGPROBS)
    a.update(kw)
    return lib.dec_sample(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(rows=-1), b"-1 rows"), (dict(rows=1 << 22), b"rows"), (dict(V=0), b"vocabulary of 0"), (dict(V=-3), b"vocabulary"),
    (dict(V=(1 << 24) + 1, stride=1 << 25), b"vocabulary"), (dict(stride=99), b"99 apart"), (dict(flags=1), b"flags"),
    (dict(x=None), b"logits"), (dict(x=P + 2), b"logits"), (dict(x=P + 1, flags=N.BF16), b"logits"),
    (dict(u=None), b"uniform"), (dict(t=P + 2), b"parameters"), (dict(k=P + 1), b"parameters"), (dict(p=P + 2), b"parameters"),
    (dict(mp=P + 2), b"parameters"), (dict(tokens=None), b"output"), (dict(tokens=P + 4), b"output"), (dict(lp=None), b"output")])
def test_sample_refuses(lib, kw, msg):
    assert sample(lib, **kw) == EINVAL and msg in lib.dec_last_error()


def test_sample_wants_its_workspace(lib):
    # 1024 sums by tiles of a row; what a part leaves: a head of 72 bytes, 2048 steps of 12, 4096 entries of 8
    def need(rows, parts):
        return rows * (8192 + parts * (72 + 2048 * 12 + 4096 * 8))
    for rows, V, top_k, flags, parts in ((64, 131072, 0, 0, 4), (1, 131072, 0, 0, 8), (1, 131072, 0, N.BF16, 4),
                                         (1, 131072, 513, 0, 8), (100, 131072, 0, 0, 2), (3, 40000, -1, 0, 2),
                                         (1, 1 << 24, 0, 0, 16)):
        assert N.sample_workspace(rows, V, top_k, flags) == need(rows, parts)
        kw = dict(rows=rows, V=V, stride=V, k=None, k_all=top_k, flags=flags)
        for more in (dict(wb=need(rows, parts) - 1), dict(work=None), dict(work=P + 8)):
            assert sample(lib, **kw, **more) == EINVAL and b"bytes of 16-byte aligned workspace" in lib.dec_last_error()
    # a part is 16 tiles of 1024 or 2048 elements at least, and there is one workgroup a compute unit; sorted lists
    # are a workgroup's
    for rows, V, top_k, flags in ((129, 131072, 0, 0), (1, 32767, 0, 0), (1, 65535, 0, N.BF16), (1, 131072, 512, 0)):
        assert N.sample_workspace(rows, V, top_k, flags) == 0
    for bad in ((-1, 10, 0, 0), (1, 0, 0, 0)):
        with pytest.raises(RuntimeError, match="sample_workspace: "):
            N.sample_workspace(*bad)


def test_nothing_to_do_needs_no_gpu(lib):
    assert conv(lib, B=0, T=0, x=None, w=None, state=None, starts=None, read=None, write=None, out=None) == 0
    assert delta(lib, B=0, T=0, q=None, k=None, v=None, state=None, starts=None, read=None, write=None, out=None,
                 work=None, wb=0) == 0
    assert sample(lib, rows=0, x=None, u=None, tokens=None, lp=None, work=None, wb=0) == 0


def test_errors_are_the_last_ones(lib):
    assert conv(lib, W=9) == EINVAL and b"causal_conv: width 9" in lib.dec_last_error()
    assert sample(lib, V=0) == EINVAL and b"sample: a vocabulary" in lib.dec_last_error()
    assert isinstance(lib.dec_last_error(), bytes) and ctypes.sizeof(ctypes.c_void_p) == 8


# ---- the functions ------------------------------------------------------------------------------
def test_tensors_must_be_on_the_gpu():
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match=r"\[radiance.decode\] causal_conv: tensors must be on the GPU"):
        G.causal_conv(bf(2, 16), bf(16, 4), None, bf(3, 3, 16), i(0, 2), i(0), i(0), 2)
    with pytest.raises(RuntimeError, match="gated_delta_rule: tensors must be on the GPU"):
        G.gated_delta_rule(bf(2, 1, 64), bf(2, 1, 64), bf(2, 1, 64), bf(2, 1), bf(2, 1), torch.zeros(1), torch.zeros(1),
                           torch.zeros(3, 1, 64, 64), i(0, 2), i(0), i(0), 2)
    with pytest.raises(RuntimeError, match="sample: tensors must be on the GPU"):
        S.sample(torch.zeros(2, 5), torch.zeros(2))


def test_fakes():
    """What a compiler sees: one opaque node each, of the right shapes."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        bf = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        i = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
        out = G.causal_conv(bf(7, 32), bf(32, 4), None, bf(3, 3, 32), i(3), i(2), i(2), 5)
        assert out.shape == (7, 32) and out.dtype == torch.bfloat16
        f = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
        out = G.gated_delta_rule(bf(7, 2, 64), bf(7, 2, 64), bf(7, 4, 128), bf(7, 4), bf(7, 4), f(4), f(4),
                                 f(3, 4, 64, 128), i(3), i(2), i(2), 5)
        assert out.shape == (7, 4, 128) and out.dtype == torch.bfloat16
        t, lp = S.sample(f(6, 50), f(6), top_k=5, logprobs=True)
        assert t.shape == lp.shape == (6,) and t.dtype == torch.int64 and lp.dtype == torch.float32
        assert S.sample(f(6, 50), f(6), temperature=f(6)).shape == (6,)


def test_states():
    s = G.new_state(2, 3, 64, 128, device="cpu", layers=4)
    assert s.shape == (4, 2, 3, 64, 128) and not s.any()
    s = G.new_conv_state(5, 48, 4, device="cpu")
    assert s.shape == (5, 3, 48) and s.dtype == torch.bfloat16
    for bad in (lambda: G.new_state(2, 3, 32, 64, "cpu"), lambda: G.new_conv_state(2, 12, 4, "cpu"),
                lambda: G.new_conv_state(2, 16, 1, "cpu")):
        with pytest.raises(RuntimeError, match="none of|multiple"):
            bad()
