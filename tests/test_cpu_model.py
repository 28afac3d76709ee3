"""Kernels of libdecode_ops.so on the CPU, over a model of a workgroup (cpu_model/), with memory that ends where the data
does: sampling as a whole, with its waves in random order; and what the convolution and the delta rule read and write, which
has to be in range whatever starts and slots hold."""
import concurrent.futures
import ctypes
import os
import re
import shutil
import subprocess
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "vllm_sly_radiance_amd", "csrc")
MODEL = os.path.join(ROOT, "tests", "cpu_model")


def compiled(tmp, name, source):
    clang = shutil.which("clang++", path=os.pathsep.join(["/opt/rocm/llvm/bin", os.environ.get("PATH", "")]))
    if not clang:
        pytest.skip("no clang++ (vector extensions)")
    path = os.path.join(tmp, name)
    with open(path + ".cpp", "w") as f:
        f.write(source)
    subprocess.run([clang, "-O1", "-g", "-std=c++17", "-fPIC", "-shared", "-w", "-fno-strict-aliasing", "-I" + MODEL, "-I" + CSRC,
                    "-I" + os.path.join(ROOT, "include"), path + ".cpp", os.path.join(MODEL, "model.cpp"), "-o",
                    path + ".so"], check=True)
    return path + ".so"


def for_cpu(name, replace=("", "")):
    """A kernel's source with its launches on the model, and the instructions that it names in plain words."""
    source = open(os.path.join(CSRC, name)).read()
    if replace[0]:
        assert source.count(replace[0]) == 1
        source = source.replace(*replace)
    source = re.sub(r"(\w+<[\w, ]+>)<<<(.+?), ([^,;]+), 0, stream>>>\(([^;]*)\);",
                    r"model::launch(\2, \3, [=] { \1(\4); });", source)
    source = re.sub(r'asm\("v_(max|min)3_f32[^;]*;', r"r = f\1(f\1(a, b), c);", source)
    assert "<<<" not in source and "asm(" not in source
    return source


SAMPLE = """
extern "C" int model_sample(const dec::SampleArgs* a) { return dec::launch_sample(*a, nullptr); }
extern "C" size_t model_workspace(int rows, int parts) { return dec::sample_workspace(rows, parts); }
extern "C" size_t model_args() { return sizeof(dec::SampleArgs); }
"""


def run(cases, library, seeds):
    def one(seed):
        return subprocess.run([sys.executable, "-u", "-m", "tests.cpu_model." + cases, library, str(seed)], cwd=ROOT,
                              capture_output=True, text=True, timeout=300)
    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        return list(pool.map(one, seeds))


def test_sampling_in_any_order_of_waves(tmp_path):
    for r in run("sample", compiled(str(tmp_path), "sample", for_cpu("dec_sample.hip") + SAMPLE), range(16)):
        assert r.returncode == 0, (r.returncode, r.stdout[-500:], r.stderr[-1500:])


@pytest.mark.parametrize("mistake", ["a missing barrier", "a read in front of the row"])
def test_the_model_shows_mistakes(tmp_path, mistake):
    """(planted in a copy for the CPU)"""
    if mistake == "a missing barrier":          # what one thread has found, read before it has left it
        old = "s.wave[wave] = mine ? x : 0, s.wave2[wave] = mine ? y : 0;\n  __syncthreads();"
        new = old.replace("\n  __syncthreads();", "")
    else:
        old, new = "if (inside || (i >= 0 && i + kRun <= V)) {", "if (inside || i + kRun <= V) {"
    library = compiled(str(tmp_path), "wrong", for_cpu("dec_sample.hip", (old, new)) + SAMPLE)
    assert any(r.returncode for r in run("sample", library, (3, 5, 6, 7)))


# ---- sequences ----------------------------------------------------------------------------------
SEQUENCES = """
namespace {
dec::Sequences sequences(const int* starts, const int* read, const int* write, int total, int batch, int max_q, int slots,
                         int cols, long slot_stride) {
  return {starts, read, write, cols ? cols : 1, slots, slot_stride, cols, total, batch, max_q};
}
}  // namespace
extern "C" int model_conv(const uint16_t* x, const uint16_t* w, uint16_t* state, const int* starts, const int* read,
                          const int* write, uint16_t* out, int total, int batch, int max_q, int slots, int cols, int C, int W) {
  dec::ConvArgs a = {};
  a.x = x, a.w = w, a.state = state, a.out = out, a.x_ts = C, a.C = C, a.silu = true;
  a.s = sequences(starts, read, write, total, batch, max_q, slots, cols, (W - 1) * C);
  return dec::launch_conv(a, W, nullptr);
}
extern "C" int model_steps(const uint16_t* q, const uint16_t* k, const uint16_t* v, const uint16_t* ga, const uint16_t* gb,
                           const float* a_log, const float* dt, float* state, const int* starts, const int* read,
                           const int* write, uint16_t* out, int total, int batch, int max_q, int slots, int cols, int Hk,
                           int Hv) {
  dec::DeltaArgs a = {};
  a.q = q, a.k = k, a.v = v, a.a = ga, a.b = gb, a.a_log = a_log, a.dt_bias = dt, a.state = state, a.out = out;
  a.q_ts = a.k_ts = Hk * 64, a.v_ts = Hv * 64, a.q_hs = a.k_hs = a.v_hs = 64, a.a_ts = a.b_ts = Hv;
  a.s = sequences(starts, read, write, total, batch, max_q, slots, cols, Hv * 64 * 64L);
  a.Hk = Hk, a.Hv = Hv, a.scale = 0.125f, a.eps = 1e-6f;
  return dec::launch_delta_steps(a, 64, 64, nullptr);
}
"""


def test_sequences_stay_in_range_whatever_the_starts_hold(tmp_path):
    source = for_cpu("dec_conv.hip") + for_cpu("dec_delta_steps.hip") + SEQUENCES
    for r in run("sequences", compiled(str(tmp_path), "sequences", source), range(8)):
        assert r.returncode == 0, (r.returncode, r.stdout[-500:], r.stderr[-1500:])


# ---- chunks of the delta rule -------------------------------------------------------------------
@pytest.fixture(scope="module")
def chunks(tmp_path_factory):
    lib = ctypes.CDLL(compiled(str(tmp_path_factory.mktemp("model")), "chunks", """
#include "dec_chunks.h"
extern "C" void model_chunks(const int* starts, int total, int batch, int slots, long* row0, int* rows, int* first, int* count) {
  using namespace dec;
  Sequences s = {};
  s.starts = starts, s.total = total, s.batch = batch;
  model::launch(slots, 64, [=] {        // as delta_prepare
    const int c = (int)blockIdx.x;
    size_t at = 0;
    int m = 0;
    const bool some = rows_of_chunk(s, c, at, m);
    if (threadIdx.x == 0) row0[c] = (long)at, rows[c] = some ? m : 0;
  });
  for (int b = 0; b < batch; ++b) {     // as delta_chunks
    int row, n;
    rows_of(s, b, row, n);
    first[b] = first_chunk(s, b), count[b] = ceil_div(n, kChunk);
  }
}
"""))

    def slots_of(starts, total):
        starts = np.ascontiguousarray(starts, np.int32)
        batch = len(starts) - 1
        slots = total // 64 + batch
        row0, rows = np.zeros(slots, np.int64), np.zeros(slots, np.int32)
        first, count = np.zeros(batch, np.int32), np.zeros(batch, np.int32)
        lib.model_chunks(*[ctypes.c_void_p(a.ctypes.data) if isinstance(a, np.ndarray) else a
                           for a in (starts, total, batch, slots, row0, rows, first, count)])
        return row0, rows, first, count, slots
    return slots_of


def test_chunks_hold_each_row_once(chunks):
    rng = np.random.default_rng(1)
    for _ in range(60):
        batch = int(rng.choice([1, 2, 5, 63, 64, 65, 130]))
        lens = rng.integers(0, rng.choice([2, 70, 300]), batch) * (rng.random(batch) < 0.8)
        total = int(lens.sum()) + int(rng.integers(0, 100))
        starts = int(rng.integers(0, total - lens.sum() + 1)) + np.concatenate([[0], np.cumsum(lens)])
        row0, rows, first, count, slots = chunks(starts, total)
        used = set()
        for b in range(batch):
            for i in range(count[b]):
                c = first[b] + i
                assert c < slots and c not in used
                used.add(c)
                assert row0[c] == starts[b] + 64 * i and rows[c] == min(lens[b] - 64 * i, 64)
        assert all(rows[c] == 0 for c in range(slots) if c not in used)


def test_chunks_stay_in_range_whatever_the_starts_hold(chunks):
    rng = np.random.default_rng(2)
    back = 0
    for _ in range(300):
        batch, total = int(rng.choice([1, 2, 3, 10, 64, 70])), int(rng.choice([1, 63, 64, 700, 5000]))
        starts = rng.integers(-10, total + 11, batch + 1)
        if rng.random() < 0.3:
            starts = rng.choice([-2 ** 31, -1, 0, total // 2, total, 2 ** 31 - 1], batch + 1)
        row0, rows, first, count, slots = chunks(starts, total)
        there = rows > 0
        assert (rows <= 64).all() and (row0[there] >= 0).all() and (row0[there] + rows[there] <= total).all()
        assert (first >= 0).all() and (first[count > 0] + count[count > 0] <= slots).all()
        back += int((np.diff(starts) < 0).any())
    assert back > 100
