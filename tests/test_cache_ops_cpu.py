"""Host side of the 8-bit cache and of shared prefixes: what needs no GPU answers without one, everything else fails loudly."""
import pytest

from distributed_inference_server_b200 import binding as B


def test_scratch_grows_with_nothing_but_its_arguments():
    lib = B.load()
    one = lib.dis_k_attn_paged_i8_scratch_elems(1, 32, 8, 128)
    assert one == lib.dis_k_attn_paged_i8_scratch_elems(1000, 32, 8, 128) > 1 << 16
    assert lib.dis_k_attn_paged_i8_scratch_elems(0, 32, 8, 128) == 0
    assert lib.dis_k_attn_paged_i8_scratch_elems(1, 0, 8, 128) == lib.dis_k_attn_paged_i8_scratch_elems(1, 32, 0, 128) == 0
    shared = [lib.dis_k_attn_shared_scratch_elems(T, 32, 8, 128) for T in (1, 2, 33, 400)]
    assert shared == sorted(shared) or shared[0] >= one
    assert all(n >= one for n in shared)
    assert lib.dis_k_attn_shared_scratch_elems(0, 32, 8, 128) == lib.dis_k_attn_shared_scratch_elems(4, 32, 0, 128) == 0


@pytest.mark.parametrize("T,nkv,d,prefix,want", [(1, 8, 128, 1 << 20, 0), (2, 8, 128, 0, 0), (32, 8, 128, 1024, 1), (32, 8, 128, 1023, 0), (64, 4, 64, 2048, 1),
                                                 (8, 4, 64, 1000, 0), (1000, 64, 128, 1 << 21, 1)])
def test_when_a_prefix_is_read_once(T, nkv, d, prefix, want):
    assert B.load().dis_k_attn_shared_in_common(T, nkv, d, prefix) == want


def test_no_cpu_fallback():
    import torch
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    lib = B.load()
    assert lib.dis_k_rope_kv_write_i8(*[None] * 1, 1, 0, *[None] * 4, 1, *[None] * 4, 1, 4, 2, 64, 16, None) == B.ERR_INFERENCE_FAILED
    assert lib.dis_k_kv_read_i8(*[None] * 5, 1, *[None] * 3, 1, 2, 64, 16, None) == B.ERR_INFERENCE_FAILED
    assert lib.dis_k_attn_paged_i8(*[None] * 4, 1, *[None] * 4, 1, 4, 2, 64, 16, None) == B.ERR_INFERENCE_FAILED
    assert lib.dis_k_attn_shared(*[None] * 3, 1, None, 1, None, None, 0, None, None, 1, 4, 2, 64, 16, None) == B.ERR_INFERENCE_FAILED
    assert b"no CPU fallback" in lib.dis_last_error()
