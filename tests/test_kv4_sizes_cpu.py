"""Which sizes an attention call over the 4-bit cache may have: as much as its kernels count, by the rows there
are and not by what they would be if every sequence had max_q of them."""
import ctypes

import pytest

from vllm_sly_radiance_amd import _native_kv4 as N


@pytest.fixture(scope="module")
def lib():
    return N.load_cdll()


def ask(lib, *sizes):
    n = ctypes.c_size_t()
    return lib.kv4_attention_workspace(*sizes, ctypes.byref(n)), n.value, lib.kv4_last_error()


@pytest.mark.parametrize("sizes", [
    # (total, batch, max_q, max_len, query heads, kv heads, d, window)
    (4607, 512, 4096, 131072, 32, 8, 128, 0),           # a chunk beside 511 decoding sequences
    (4351, 256, 4096, 131072, 48, 16, 128, 0),
    (17407, 1024, 16384, 131072, 128, 8, 128, 0),
    (8703, 512, 8192, 1 << 20, 64, 8, 256, 0),
    (4096, 4096, 1, 131072, 64, 8, 128, 0),
    (16, 16, 1, 0x7FFFF000, 64, 8, 128, 0),
    (64, 8, 8, 1 << 22, 64, 8, 128, 0),
    (65536, 16, 4096, 131072, 128, 128, 64, 4096),
    (1, 1, 1 << 30, 131072, 32, 8, 128, 0)])            # a limit on the queries far above the rows
def test_served(lib, sizes):
    rc, workspace, error = ask(lib, *sizes)
    assert rc == 0, error
    assert workspace < 1 << 30


def test_a_limit_above_the_rows_is_the_rows(lib):
    for total, batch, max_len, d in ((40, 3, 9000, 128), (700, 1, 5000, 256), (900, 4, 3000, 64)):
        sizes = (max_len, 32, 8, d, 0)
        assert ask(lib, total, batch, total, *sizes)[1] == ask(lib, total, batch, 1 << 20, *sizes)[1]


@pytest.mark.parametrize("sizes,msg", [
    ((1 << 22, 1 << 22, 1, 131072, 64, 8, 128, 0), b"too much"),        # 2^35 granules of 128 tokens
    ((17, 17, 1, 0x7FFFF000, 64, 8, 128, 0), b"too much"),
    ((1 << 24, 1 << 24, 1, 1, 64, 8, 128, 0), b"too much"),             # 2^27 workgroups of 512 threads
    ((1 << 25, 1 << 12, 1 << 13, 1 << 13, 64, 64, 128, 0), b"too much"),
    ((1 << 30, 8, 1 << 30, 4096, 16, 16, 64, 0), b"too many rows"),
    ((3, 1 << 30, 3, 4096, 4, 2, 64, 0), b"too many rows"),
    ((3, 1 << 20, 1 << 20, 4096, 4, 2, 64, 0), b"too many rows"),
    ((2**31 - 1, 2**31 - 1, 2**31 - 1, 4096, 4096, 4096, 64, 0), b"too many rows")])
def test_refused(lib, sizes, msg):
    rc, _, error = ask(lib, *sizes)
    assert rc == 1 and msg in error, error


def test_rows_under_a_limit_of_no_queries_are_not_nothing_to_do(lib):
    """Their outputs have to be written (NaN), so that the call needs its tensors."""
    call = lambda total: lib.kv4_attention(  # noqa: E731
        None, 0, 0, None, 0, 17 * 128, 16, None, 0, 0, None, None, None, None, 0, total, 2, 0, 10, 2, 1, 128,
        1.0, 0, 0, None)
    assert call(0) == 0
    assert call(5) == 1 and b"null q" in lib.kv4_last_error()
