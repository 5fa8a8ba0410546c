"""Keys and values in 8 bits and attention of shared prefixes at the edges of what their entries take: starts that are only as aligned as the header
asks, more rows than one launch holds, one key that leads far in front of a long flat history.  Bounds as in tests/test_cache_ops_gpu.py."""
import numpy as np
import pytest
import torch

from tests import _gpu_util as G
from tests._gpu_util import DEV, check, dev_i32, lib, ptr, sync
from tests.test_cache_ops_gpu import Cache, attention, decode, near, queries, scratch, shared
from tests.test_cache_ops_gpu import test_write_and_read as write_and_read

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ read-back
@pytest.mark.parametrize("d,page,off", [(64, 16, 8), (128, 64, 8), (128, 8, 24), (64, 32, 16)])
def test_read_into_a_pool_that_starts_on_16_bytes(d, page, off):
    """The bf16 pool starts `off` entries behind a 256-byte boundary: on 16 bytes as the header asks, and only off = 16 on 32."""
    ctx, nkv = [1, 100, page, 0, 3 * page + 5], 3
    c = Cache(ctx, nkv, d, page, 7)
    area = G.empty((c.n_pages * 2 * nkv * page * d + 32,), torch.bfloat16)
    area.zero_()
    back = area[off:off + c.n_pages * 2 * nkv * page * d].view(c.n_pages, 2, nkv, page, d)
    assert back.data_ptr() % 16 == 0 and (back.data_ptr() % 32 == 0) == (off % 16 == 0)
    check(lib().dis_k_kv_read_i8(ptr(c.pool), ptr(c.scale), ptr(back), ptr(c.d_table), ptr(c.d_table), c.width, ptr(dev_i32(np.arange(len(ctx)))), None,
                                 ptr(dev_i32(ctx)), len(ctx), nkv, d, page, None))
    sync()
    used = c.used.to(DEV)[:, None, None, :, None].expand(back.shape)
    want = torch.where(used, c.value.float().to(torch.bfloat16), torch.zeros((), dtype=torch.bfloat16, device=DEV))
    assert torch.equal(back, want)
    assert int((area[:off] != 0).sum()) == 0 and int((area[off + back.numel():] != 0).sum()) == 0


# ------------------------------------------------------------------------------------------------ a leading key and a long flat history
class Flat(Cache):
    """Histories whose first key leads for a query along dimension 0; all others score 0 there.  Its value is 1 in dimension 0 and 0 elsewhere, theirs are
    random with a largest entry of 1: every other dimension of the result is the sum of many weights, each a tiny part of the first."""

    def __init__(self, ctx, nkv, d, page, seed, common=0):
        super().__init__(ctx, nkv, d, page, seed, True, common, spread=False, amp=self.rows_of)

    def rows_of(self, x, g):
        v = torch.rand(x.shape, generator=g, device=DEV) * 0.5 + 0.5
        v[:, 0, ..., 0] = 0.0
        v[:, 1, ..., 1] = 1.0
        for b in range(self.table.shape[0]):
            if self.ctx[b] > 0:
                first = int(self.table[b, 0])
                v[first, :, :, 0] = 0.0
                v[first, :, :, 0, 0] = 1.0
        return v / torch.where(x == 0, 1.0, x)  # (the base multiplies its normal numbers by this)


def along_0(T, nh, d, size):
    q = torch.zeros(T, nh, d, device=DEV)
    q[:, :, 0] = size
    return G._guarded_copy(q.view(T, nh * d).to(torch.bfloat16))


def flat_bound(c, q, nh):
    """As `attention` bounds 8-bit pages, with the products' smallest step at 2^-32 of the largest."""
    c.int8 = False  # (its own term is 2^-25)
    o, tol = attention(c, q, nh, 2.0 ** -11)
    c.int8 = True
    for t in range(q.shape[0]):
        k, v = c.rows(t)
        p = torch.softmax(q[t].double().view(c.nkv, nh // c.nkv, c.d) @ k.transpose(1, 2) / c.d ** 0.5, -1)
        vs = (v.abs().amax(-1) / 127)[:, None]
        whole = (v / vs[..., 0, :, None]).abs().sum(1)[:, None]
        tol[t] += (2.0 ** -32 * (p * vs).amax(-1, keepdim=True) * whole).reshape(nh, c.d)
    return o, tol


def test_decode_many_small_weights_behind_a_large_one():
    """The others' weights are 2^-25.2 of the first's (140 / sqrt(64) / ln 2).  32 tiles of a history lie in one or two CTAs."""
    c = Flat([512] * 512, 1, 64, 64, 3)
    q = along_0(512, 1, 64, 140.0)
    near(decode(c, q, 1), flat_bound(c, q, 1))


def test_shared_prefix_many_small_weights_behind_a_large_one():
    T, nkv, prefix = 40, 32, 512
    assert lib().dis_k_attn_shared_in_common(T, nkv, nkv, 64, prefix, 1) == 1
    c = Flat([prefix + 1 + t % 5 for t in range(T)], nkv, 64, 64, 4, prefix)
    q = along_0(T, nkv, 64, 140.0)
    near(shared(c, q, nkv, prefix), flat_bound(c, q, nkv))


# ------------------------------------------------------------------------------------------------ weights of a shared prefix
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T,group,nkv,d,page,prefix", [(32, 4, 8, 128, 64, 2000), (70, 4, 8, 128, 16, 1501), (130, 1, 8, 64, 64, 1400), (80, 8, 8, 64, 32, 1001)])
def test_shared_prefix_weights(int8, T, group, nkv, d, page, prefix):
    """Weights enter the product as two bf16 halves (2^-16 of a weight) over bf16 pages, in fp16 (2^-11) over 8-bit ones, read once or not."""
    assert lib().dis_k_attn_shared_in_common(T, nkv * group, nkv, d, prefix, int8) == 1
    ctx = [prefix + 1 + 3 * t % 60 for t in range(T)]
    c = Cache(ctx, nkv, d, page, T + d, int8, prefix)
    q = queries(T, nkv * group, d, 61)
    out = shared(c, q, nkv * group, prefix)
    near(out, attention(c, q, nkv * group, 2.0 ** -11 if int8 else 2.0 ** -16))


# ------------------------------------------------------------------------------------------------ many tokens
@pytest.mark.parametrize("T", [125, 126, 300, 600])
@pytest.mark.parametrize("int8", [False, True])
def test_many_tokens_alone(int8, T):
    """Every token by itself, around the number of tokens from which fewer CTAs of heads of 128 over bf16 pages are resident, and past one launch's 512."""
    prefix, nkv, group = 20, 2, 4
    ctx = [prefix + int(v) for v in np.random.default_rng(T).integers(0, 150, T)]
    ctx[0], ctx[5], ctx[T - 1] = prefix + 150, 0, 7
    assert lib().dis_k_attn_shared_in_common(T, nkv * group, nkv, 128, prefix, int8) == 0
    c = Cache(ctx, nkv, 128, 16, T, int8, prefix)
    q = queries(T, nkv * group, 128, 62)
    near(shared(c, q, nkv * group, prefix), attention(c, q, nkv * group, 2.0 ** -11 if int8 else 2.0 ** -16))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T,group,nkv,d", [(520, 1, 8, 64), (1030, 4, 4, 128)])
def test_many_tokens_with_a_prefix_read_once(int8, T, group, nkv, d):
    """More tokens than one launch of the own parts takes: the prefix's kernel starts behind the last of them."""
    prefix = 333
    assert lib().dis_k_attn_shared_in_common(T, nkv * group, nkv, d, prefix, int8) == 1
    ctx = [prefix + int(v) for v in np.random.default_rng(T).integers(0, 40, T)]
    ctx[3], ctx[513], ctx[T - 1] = 0, prefix - 1, prefix
    c = Cache(ctx, nkv, d, 16, T, int8, prefix)
    q = queries(T, nkv * group, d, 63)
    area = scratch(T, nkv * group, nkv, d, True)
    out = shared(c, q, nkv * group, prefix, area=area)
    near(out, attention(c, q, nkv * group, 2.0 ** -11 if int8 else 2.0 ** -16))
    area[1 << 16:].fill_(3.0)
    assert torch.equal(shared(c, q, nkv * group, prefix, area=area), out)


def test_read_back_of_more_rows_than_one_launch():
    rows, nkv, d, page = 2100, 1, 64, 8
    ctx = [int(v) for v in np.random.default_rng(5).integers(0, 20, rows)]
    first = [int(v) for v in np.random.default_rng(6).integers(0, 12, rows)]
    c = Cache(ctx, nkv, d, page, 8)
    back = G.zeros((c.n_pages, 2, nkv, page, d), torch.bfloat16)
    check(lib().dis_k_kv_read_i8(ptr(c.pool), ptr(c.scale), ptr(back), ptr(c.d_table), ptr(c.d_table), c.width, ptr(dev_i32(np.arange(rows))), ptr(dev_i32(first)),
                                 ptr(dev_i32(ctx)), rows, nkv, d, page, None))
    sync()
    want = torch.zeros_like(back)
    for b in range(rows):
        pos = np.arange(first[b], ctx[b])
        if len(pos):
            at, slot = torch.from_numpy(c.table[b, pos // page].astype(np.int64)).to(DEV), torch.from_numpy(pos % page).to(DEV)
            want[at, :, :, slot] = c.value[at, :, :, slot].float().to(torch.bfloat16)
    assert torch.equal(back, want)


# ------------------------------------------------------------------------------------------------ writing
@pytest.mark.parametrize("nh,nkv,d,page,S,lens", [(32, 8, 128, 64, 1, [700, 300]), (32, 4, 64, 16, 3, [500, 1, 90]), (8, 8, 128, 16, 4, [800]), (64, 8, 128, 32, 2, [148])])
def test_write_of_many_tokens(nh, nkv, d, page, S, lens):
    """More CTAs than five an SM: the variant that keeps eight of them there."""
    rows = 256 // (d // 8)
    assert sum(lens) * -(-(nh + 2 * nkv) // rows) >= 5 * 148
    write_and_read(nh, nkv, d, page, S, lens)
