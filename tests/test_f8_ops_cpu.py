"""Host side of the products in 8-bit floating point: without a GPU everything fails loudly, and a shape's engine flag is a flag of its own."""
import pytest

from distributed_inference_server_b200 import binding as B


def test_no_cpu_fallback():
    import torch
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    lib = B.load()
    assert lib.dis_k_quant_f8(None, None, None, 1, 128, None) == B.ERR_INFERENCE_FAILED
    assert lib.dis_k_quant_weight_f8(None, None, None, 1, 128, None) == B.ERR_INFERENCE_FAILED
    assert lib.dis_k_add_rmsnorm_f8(*[None] * 4, 0, 0, *[None] * 4, 1, 128, 1e-5, None) == B.ERR_INFERENCE_FAILED
    assert lib.dis_k_gemm_f8(*[None] * 5, B.F32, 1, 16, 128, None) == B.ERR_INFERENCE_FAILED
    assert lib.dis_k_gemm_silu_f8(*[None] * 6, 1, 16, 128, None) == B.ERR_INFERENCE_FAILED
    assert lib.dis_k_ffn_f8(*[None] * 10, B.F32, 1, 128, 128, None) == B.ERR_INFERENCE_FAILED
    assert b"no CPU fallback" in lib.dis_last_error()


def test_engine_flags_are_distinct_bits():
    flags = [B.FLAG_NO_GRAPH, B.FLAG_FORCE_GEMV, B.FLAG_NO_PDL, B.FLAG_PREFIX_CACHE, B.FLAG_KV_INT8, B.FLAG_ATTN_SHARED, B.FLAG_WEIGHTS_F8]
    assert sorted(flags) == [1 << i for i in range(len(flags))]
