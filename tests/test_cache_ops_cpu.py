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


@pytest.mark.parametrize("T,nh,nkv,d,prefix,int8,want", [
    (1, 32, 8, 128, 1 << 20, 0, 0), (2, 32, 8, 128, 0, 0, 0), (32, 32, 8, 128, 1024, 0, 1), (32, 32, 8, 128, 1023, 0, 0), (64, 32, 4, 64, 2048, 1, 1),
    (8, 32, 4, 64, 1000, 0, 0), (1000, 64, 64, 128, 1 << 21, 1, 1), (32, 32, 8, 128, 1279, 1, 0), (32, 32, 8, 128, 1280, 1, 1), (33, 32, 8, 128, 1241, 0, 0),
    (33, 32, 8, 128, 1242, 0, 1), (64, 64, 8, 128, 767, 1, 0), (64, 64, 8, 128, 768, 1, 1), (4, 0, 0, 128, 1 << 20, 0, 0), (5, 32, 8, 128, 1 << 20, 1, 0),
    (6, 32, 8, 128, 6827, 1, 1), (2, 32, 8, 128, 32767, 0, 0), (2, 32, 8, 128, 32768, 0, 1), (4, 32, 8, 128, 8192, 0, 1)])
def test_when_a_prefix_is_read_once(T, nh, nkv, d, prefix, int8, want):
    assert B.load().dis_k_attn_shared_in_common(T, nh, nkv, d, prefix, int8) == want


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
