"""Sizes that the calls on 8-bit floating point refuse: checked before anything else, so that it shows without a GPU too."""
import pytest

from distributed_inference_server_b200 import binding as B

MOST_T, MOST_N, MOST_K = 65535 * 32, 65535 * 128, 1 << 30


def calls(T, N, K):
    """Each entry with T rows of K entries and a weight of N rows, where it has them: (its name, what it returns)"""
    lib = B.load()
    yield "quant_f8", lib.dis_k_quant_f8(None, None, None, T, K, None)
    yield "quant_weight_f8", lib.dis_k_quant_weight_f8(None, None, None, N, K, None)
    yield "add_rmsnorm_f8", lib.dis_k_add_rmsnorm_f8(*[None] * 4, 0, 0, *[None] * 4, T, K, 1e-5, None)
    yield "gemm_f8", lib.dis_k_gemm_f8(*[None] * 5, B.F32, T, N, K, None)
    yield "gemm_silu_f8", lib.dis_k_gemm_silu_f8(*[None] * 6, T, N, K, None)
    yield "ffn_f8", lib.dis_k_ffn_f8(*[None] * 10, B.F32, T, K, N, None)


@pytest.mark.parametrize("K", [MOST_K + 16, 2147483536, 2147483632, -16, 0, 8, 24])
def test_rows_of_other_lengths(K):
    for name, rc in calls(1, 16, K):
        assert rc == B.ERR_INVALID_ARGUMENT, name


@pytest.mark.parametrize("T", [MOST_T + 1, -1])
def test_more_rows(T):
    for name, rc in calls(T, 16, 128):
        if name != "quant_weight_f8":  # (it has none)
            assert rc == B.ERR_INVALID_ARGUMENT, name


@pytest.mark.parametrize("N", [MOST_N + 16, -16])
def test_more_rows_of_a_weight(N):
    for name, rc in calls(1, N, 128):
        if name not in ("quant_f8", "add_rmsnorm_f8"):
            assert rc == B.ERR_INVALID_ARGUMENT, name


@pytest.mark.parametrize("K", [2147483536, MOST_K + 16])
def test_a_refusal_says_what(K):
    assert B.load().dis_k_quant_f8(None, None, None, 1, K, None) == B.ERR_INVALID_ARGUMENT
    assert b"2^30" in B.load().dis_last_error()
