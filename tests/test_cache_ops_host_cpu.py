"""Host side of shared prefixes: which batches read a prefix once, and how large the scratch is."""
import pytest

from distributed_inference_server_b200 import binding as B


@pytest.mark.parametrize("T,nh,nkv,want", [(65535 * 128, 8, 8, 1), (65535 * 128 + 1, 8, 8, 0), (65535 * 16, 64, 8, 1), (65535 * 16 + 1, 64, 8, 0), (1 << 30, 8, 8, 0), (0x7fffffff, 64, 8, 0),
                                           (64, 65535, 65535, 1), (64, 65536, 65536, 0)])
def test_batches_that_no_grid_holds_go_alone(T, nh, nkv, want):
    """More than 65535 tiles of 128 rows, or kv heads, are not refused: every token goes alone."""
    assert B.load().dis_k_attn_shared_in_common(T, nh, nkv, 128, 4096, 0) == want


@pytest.mark.parametrize("nh,nkv,d", [(32, 8, 128), (8, 8, 64), (64, 8, 128), (32, 4, 64)])
def test_scratch_holds_what_a_call_keeps(nh, nkv, d):
    """The pieces' part, every token's own state, and a state per 128-row tile, kv head and slice, of which there is at least one."""
    lib = B.load()
    pieces = lib.dis_k_attn_paged_i8_scratch_elems(1, nh, nkv, d)
    group = nh // nkv
    for T in (1, 2, 31, 32, 33, 128, 400, 5000):
        tiles = -(-T * group // 128)
        blocks = (tiles if tiles < 2 else (tiles + 1) // 2) * nkv
        slices = min(32, max(1, 2 * 148 // blocks))
        need = pieces + T * nh * (d + 2) + slices * nkv * tiles * 128 * (d + 2)
        assert need <= lib.dis_k_attn_shared_scratch_elems(T, nh, nkv, d) <= need + 8
