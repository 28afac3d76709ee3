"""Sizes at which indexes of libdecode_ops.so would leave their range are refused (no GPU is used)."""
import pytest

from tests.test_decode_abi_cpu import EINVAL, conv, delta, lib  # noqa: F401


def run_starts(total, max_q, blocks=1, batch=1):
    """Where a lane of the convolution begins its runs of 16 tokens, the first and the ones it takes after it
    (dec_conv.hip, conv_rows and launch_conv): the largest that is formed for a sequence of all tokens."""
    grid = (1 << 32) // 256 - 1
    runs = min(max(-(-min(max_q, total) // 16), 1), max(grid // blocks // batch, 1))
    step = runs * 16
    return (total - 1) // step * step + step + (runs - 1) * 16


def test_runs_of_the_longest_sequences_are_counted_in_32_bits():
    most = 1 << 30
    for max_q in (1, 17, 1000, 1 << 20, 1 << 28, most):
        for blocks in (1, 8192):
            for total in (1, 16, 4097, most - 1, most):
                assert run_starts(total, max_q, blocks) < 2 ** 31
    assert run_starts(2 ** 31 - 1, 2 ** 31 - 1) >= 2 ** 31          # why there is a limit


@pytest.mark.parametrize("T", [(1 << 30) + 1, (1 << 31) - 1])
def test_conv_of_more_tokens_is_refused(lib, T):  # noqa: F811
    assert conv(lib, T=T, C=8, ts=8, ss=24, mq=T, B=1) == EINVAL and b"2^30 at most" in lib.dec_last_error()


def test_delta_rule_of_as_many_is_too_large(lib):  # noqa: F811
    assert delta(lib, T=(1 << 30) + 1, Hk=1, Hv=1, ss=128 * 128, B=1) == EINVAL and b"too large" in lib.dec_last_error()


def test_rows_with_a_top_k_of_their_own_are_one_part():
    """(dec_sample.hip relies on it: of rows in parts none goes by a sorted list)"""
    from vllm_sly_radiance_amd import _native_decode as N
    for rows in (1, 2, 64, 300):
        for V in (1, 2, 511, 512, 513, 32768, 131072, 1 << 24):
            for flags in (0, N.BF16, N.LOGPROBS):
                assert N.sample_workspace(rows, V, 1, flags) == 0
                for k in (1, 50, 512):
                    assert N.sample_workspace(rows, V, k, flags) == 0 or k >= V


def test_workspace_of_the_chunks_is_as_documented():
    from vllm_sly_radiance_amd import _native_decode as N
    for total, batch, Hk, Hv, dk, dv in ((4001, 1, 16, 48, 128, 128), (30000, 16, 8, 16, 64, 64), (63, 2, 1, 4, 64, 128)):
        need = (total // 64 + batch) * (25600 * Hv + (49152 if dk == 128 else 24576) * Hk)
        assert N.gated_delta_workspace(total, batch, 17, 0, Hk, Hv, dk, dv) == need
        for max_q, cols in ((16, 0), (17, 1)):
            assert N.gated_delta_workspace(total, batch, max_q, cols, Hk, Hv, dk, dv) == 0
