"""Build libw4a8_mxfp4.so and libkv4_attn.so in-tree with hipcc for gfx950 (no other target), and
_kv4_torch.so, the latter's binding to torch tensors, with the host compiler.

    python -m vllm_sly_radiance_amd.build            # or __graft_entry__.build()

The libraries are plain C-ABI shared objects (include/w4a8_mxfp4.h, include/kv4_attn.h) loaded
through ctypes; they link the HIP runtime by soname, so inside a torch process they bind to the
runtime torch already loaded. _kv4_torch.so is a CPython module over libkv4_attn.so, built against the
installed torch's headers.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB_NAME = "libw4a8_mxfp4.so"
LIB_PATH = os.path.join(PKG, LIB_NAME)
ARCH = "gfx950"

SOURCES = ["w4a8_api.hip", "w4a8_quant.hip", "w4a8_repack.hip", "w4a8_gemm_skinny.hip",
           "w4a8_gemm_stream.hip", "w4a8_gemm_ring.hip", "w4a8_gemm_tile.hip", "w4a8_gemm_band.hip",
           "w4a8_producers.hip", "w4a8_probe.hip"]

KV4_LIB_PATH = os.path.join(PKG, "libkv4_attn.so")
KV4_SOURCES = ["kv4_api.hip", "kv4_rope.hip", "kv4_pages.hip", "kv4_attn_rows.hip",
               "kv4_attn_tiles.hip"]
KV4_TORCH_PATH = os.path.join(PKG, "_kv4_torch.so")
KV4_TORCH_SOURCE = "kv4_torch.cpp"

FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
    # keep the compiler from forming packed-fp32 VALU ops (v_pk_*_f32)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # the first 14 kernel-argument dwords arrive in SGPRs at wave launch instead of through a
    # scalar load from the kernarg segment (the kernels order their arguments so that everything
    # the first memory requests depend on comes first); the code object keeps a 256-byte prologue
    # that loads them itself where the firmware does not preload
    "-mllvm", "-amdgpu-kernarg-preload-count=14",
    "-Wall", "-Wno-unused-function",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (expected /opt/rocm/bin/hipcc)")


def _command(sources, out) -> list[str]:
    srcs = [os.path.join(CSRC, s) for s in sources]
    return [hipcc(), *FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", *srcs, "-o", out]


def _torch_commands(out) -> tuple[list[str], list[str]]:
    """Compile and link the torch binding (the link needs libkv4_attn.so, found again beside it)."""
    import torch
    base = os.path.dirname(torch.__file__)
    cxx = os.environ.get("CXX") or "g++"
    system = [os.path.join(base, "include"), "/opt/rocm/include", sysconfig.get_paths()["include"]]
    compile_ = [cxx, "-c", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-Wall",
                "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
                f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f"-I{INCLUDE}",
                *(a for d in system for a in ("-isystem", d)),
                os.path.join(CSRC, KV4_TORCH_SOURCE), "-o", out + ".o"]
    link = [cxx, "-shared", out + ".o", "-o", out, f"-L{PKG}", "-l:" + os.path.basename(KV4_LIB_PATH),
            f"-L{os.path.join(base, 'lib')}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python",
            "-Wl,-rpath,$ORIGIN"]
    return compile_, link


def _run(cmd, verbose):
    """The command's process, started."""
    if verbose:
        print(" ".join(cmd), flush=True)
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def _end(job, verbose) -> None:
    """Waits for a compiler; RuntimeError with its words where it failed."""
    text = job.communicate()[0]
    # hipcc's host pass does not know the packed-fp32 target feature; that warning is expected
    noise = [ln for ln in text.splitlines()
             if ln.strip() and "packed-fp32-ops" not in ln and "warning generated" not in ln
             and "warnings generated" not in ln]
    if job.returncode != 0:
        raise RuntimeError("the compiler failed:\n" + "\n".join(noise))
    if verbose and noise:
        print("\n".join(noise), file=sys.stderr)


def build(verbose: bool = False) -> str:
    """Compile every source into LIB_PATH, KV4_LIB_PATH and KV4_TORCH_PATH (always rebuilds, all at
    once) and return LIB_PATH. What compiles is put in place whatever becomes of the rest: the linear
    path's library needs hipcc only. RuntimeError at the end where something did not."""
    libraries = [(path, _run(_command(sources, path + ".tmp"), verbose))
                 for sources, path in ((SOURCES, LIB_PATH), (KV4_SOURCES, KV4_LIB_PATH))]
    tmp, errors, link = KV4_TORCH_PATH + ".tmp", [], None
    try:
        compile_, link = _torch_commands(tmp)
        binding = _run(compile_, verbose)
    except (OSError, ImportError, AttributeError) as e:        # no host compiler, no torch or not its headers
        binding, link = None, None
        errors.append(f"_kv4_torch cannot be built: {e}")
    for path, job in libraries:
        try:
            _end(job, verbose)
            os.replace(path + ".tmp", path)
        except RuntimeError as e:
            errors.append(str(e))
            if path == KV4_LIB_PATH:
                link = None
    try:
        if binding:
            _end(binding, verbose)
            if link:
                _end(_run(link, verbose), verbose)
                os.replace(tmp, KV4_TORCH_PATH)
            os.remove(tmp + ".o")
    except RuntimeError as e:
        errors.append(str(e))
    if errors:
        raise RuntimeError("\n".join(errors))
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose=True))
