"""Keys and values in 8 bits (written, read back, attended over) and attention of a shared prefix, through the C ABI, against the definitions in
64 bits.  Every bound follows from the roundings that the operators make:
  a bf16 result        eight significant bits: half a unit in the last place is at most 2^-8 of it;
  8-bit rows           half a step of the row's scale;
  a score              fp32 sums of d products, 2^-20 of sum |q k| / sqrt(d), which moves a weight by as much (relatively);
  a weight             2^-11 of it in fp16 (8-bit pages), 2^-8 in bf16, and the weights' sum moves likewise: twice that times sum p |v|;
                       fp16 has no numbers between multiples of 2^-24: 2^-25 of the largest p vs (vs: the values' scale) times sum |v8|.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from distributed_inference_server_b200 import binding as B
from tests import _gpu_util as G
from tests._gpu_util import DEV, check, dev_i32, lib, ptr, sync

pytestmark = pytest.mark.gpu
NAN = float("nan")


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def guarded(t):
    x = G.empty(t.shape, t.dtype)
    x.copy_(t)
    return x


def scratch(T, nh, nkv, d, shared=False):
    n = (lib().dis_k_attn_shared_scratch_elems if shared else lib().dis_k_attn_paged_i8_scratch_elems)(T, nh, nkv, d)
    return G.zeros(n)


def quantise(x):
    """Rows of x in 8 bits: whole numbers, scales."""
    s = x.abs().amax(-1) / 127
    return torch.round(x / torch.where(s > 0, s, 1.0)[..., None]).to(torch.int8), s.float()


class Cache:
    """A paged pool of histories of ctx[b] tokens (pages in shuffled order).  The first `common` positions of all rows hold the same: whole pages of them
    are the same pages, of a page in which they end every row has a copy.  Rows that no history covers hold 8-bit noise and NaN scales (bf16: zeros
    in pages of the prefix, NaN elsewhere), table entries without a page are far out of range."""

    def __init__(self, ctx, nkv, d, page, seed, int8=True, common=0, spread=True, width=None, amp=None):
        g, r = gen(seed), np.random.default_rng(seed)
        self.nkv, self.d, self.page, self.int8, self.ctx = nkv, d, page, int8, list(ctx)
        pages = [max(0, -(-c // page)) for c in ctx]
        if common:
            pages[0] = max(pages[0], -(-common // page))  # the first row's pages hold the whole prefix
        shared = common // page
        n_pages = shared + sum(max(0, p - shared) for p in pages) + 1
        order = r.permutation(n_pages)
        self.width = width or max(max(pages), 1) + 2
        table = np.full((len(ctx), self.width), 1 << 29, np.int32)
        at = shared
        for b, p in enumerate(pages):
            k = max(0, p - shared)
            table[b, :min(p, shared)] = order[:min(p, shared)]
            table[b, shared:shared + k] = order[at:at + k]
            at += k
        self.table, self.n_pages = table, n_pages
        x = torch.randn(n_pages, 2, nkv, page, d, generator=g, device=DEV)
        if spread:
            x = x * (torch.rand(n_pages, 2, nkv, page, 1, generator=g, device=DEV) + 0.5)
        if amp is not None:
            x = x * amp(x, g)
        if common % page:  # every row's copy of the prefix's end
            first = int(table[0, shared])
            for b in range(1, len(ctx)):
                if pages[b] > shared:
                    x[int(table[b, shared]), :, :, :common % page] = x[first, :, :, :common % page]
        self.used = torch.zeros(n_pages, page, dtype=torch.bool)
        for b, c in enumerate(ctx):
            for i in range(pages[b]):
                self.used[table[b, i], :max(0, min(page, c - i * page))] = True
        if common:
            for i in range(pages[0]):
                self.used[table[0, i], :max(0, min(page, common - i * page))] = True
        hidden = ~self.used.to(DEV)
        if int8:
            q, s = quantise(x)
            s.masked_fill_(hidden[:, None, None, :], NAN)
            self.pool, self.scale = guarded(q), guarded(s)
            self.value = q.double() * s.double()[..., None]
        else:
            v = x.to(torch.bfloat16)
            v = torch.where(hidden[:, None, None, :, None], torch.tensor(NAN, dtype=torch.bfloat16, device=DEV), v)
            for i in range(-(-common // page)):  # rows behind the prefix in its last page are finite, as the contract asks
                v[int(table[0, i])] = torch.nan_to_num(v[int(table[0, i])])
            self.pool, self.scale = guarded(v), None
            self.value = v.double()
        self.d_table = dev_i32(table)

    def rows(self, b):
        """K and V [nkv][ctx][d] of history b in 64 bits."""
        n = max(0, self.ctx[b])
        p = self.table[b, :-(-n // self.page)].astype(np.int64)
        kv = self.value[torch.from_numpy(p).to(DEV)].permute(1, 2, 0, 3, 4).reshape(2, self.nkv, -1, self.d)[:, :, :n]
        return kv[0], kv[1]


def attention(cache, q, nh, weight_err):
    """(result, bound) [T][nh][d] in 64 bits."""
    T, d = q.shape[0], cache.d
    group = nh // cache.nkv
    out, tol = torch.zeros(T, nh, d, dtype=torch.float64, device=DEV), torch.zeros(T, nh, d, dtype=torch.float64, device=DEV)
    for t in range(T):
        if cache.ctx[t] <= 0:
            continue
        k, v = cache.rows(t)
        qt = q[t].double().view(cache.nkv, group, d)
        p = torch.softmax(qt @ k.transpose(1, 2) / math.sqrt(d), -1)
        o, a = p @ v, p @ v.abs()
        size = (qt.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) / math.sqrt(d)
        out[t] = o.reshape(nh, d)
        tol[t] = (2.0 ** -8 * o.abs() + 2 * (weight_err + 2.0 ** -20 * size) * a + 1e-30).reshape(nh, d)
        if cache.int8:
            vs = (v.abs().amax(-1) / 127)[:, None]
            whole = (v / torch.where(vs > 0, vs, 1.0)[..., 0, :, None]).abs().sum(1)[:, None]
            tol[t] += (2.0 ** -25 * (p * vs).amax(-1, keepdim=True) * whole).reshape(nh, d)
    return out, tol


def decode(cache, q, nh, stream=None, area=None, rows=None):
    T = q.shape[0]
    out = G.empty((T, nh * cache.d), torch.bfloat16)
    area = scratch(T, nh, cache.nkv, cache.d) if area is None else area
    rows = dev_i32(np.arange(T)) if rows is None else rows
    check(lib().dis_k_attn_paged_i8(ptr(q), ptr(cache.pool), ptr(cache.scale), ptr(cache.d_table), cache.width, ptr(rows), ptr(dev_i32(cache.ctx)),
                                    ptr(out), ptr(area), T, nh, cache.nkv, cache.d, cache.page, stream))
    sync()
    n = area.numel()
    assert int((area.view(torch.int32)[:min(n, 1 << 16)] != 0).sum()) == 0  # as the next call wants it
    return out


def shared(cache, q, nh, prefix, stream=None, area=None):
    T = q.shape[0]
    out = G.empty((T, nh * cache.d), torch.bfloat16)
    area = scratch(T, nh, cache.nkv, cache.d, True) if area is None else area
    check(lib().dis_k_attn_shared(ptr(q), ptr(cache.pool), ptr(cache.scale), cache.n_pages, ptr(cache.d_table), cache.width,
                                  ptr(dev_i32(np.arange(T))), ptr(dev_i32(cache.ctx)), prefix, ptr(out), ptr(area), T, nh, cache.nkv, cache.d, cache.page,
                                  stream))
    sync()
    return out


def queries(T, nh, d, seed, size=1.5):
    return guarded((torch.randn(T, nh * d, generator=gen(seed + 1000), device=DEV) * size).to(torch.bfloat16))


def near(out, want):
    o, tol = want
    got = out.double().view(o.shape)
    bad = (got - o).abs() - tol
    assert torch.isfinite(got).all()
    assert float(bad.max()) <= 0, (float((got - o).abs().max()), [int(v) for v in np.unravel_index(int(bad.argmax()), o.shape)])


# ------------------------------------------------------------------------------------------------ attention over 8-bit pages
RAGGED = [0, 1, 15, 16, 17, 31, 33, 64, 65, 127, 128, 129, 300, 1000]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 4, 8])
@pytest.mark.parametrize("nkv,page", [(1, 64), (3, 8), (8, 16)])
def test_decode_ragged(d, group, nkv, page):
    c = Cache(RAGGED, nkv, d, page, d + group + nkv)
    q = queries(len(RAGGED), nkv * group, d, group)
    out = decode(c, q, nkv * group)
    near(out, attention(c, q, nkv * group, 2.0 ** -11))
    assert int((out[0] != 0).sum()) == 0  # no keys: zeros


@pytest.mark.parametrize("ctx", [[1], [5000], [20000, 3], [7, 4099, 2000, 2000, 900, 1, 1, 6001], [40] * 300, [0, 0, 0], [0] * 5 + [33]])
def test_decode_lengths(ctx):
    c = Cache(ctx, 2, 128, 32, 11)
    q = queries(len(ctx), 8, 128, 12)
    near(decode(c, q, 8), attention(c, q, 8, 2.0 ** -11))


def test_decode_more_tokens_than_one_launch():
    ctx = [int(v) for v in np.random.default_rng(0).integers(0, 40, 1100)]
    c = Cache(ctx, 1, 64, 16, 13)
    q = queries(len(ctx), 1, 64, 14)
    near(decode(c, q, 1), attention(c, q, 1, 2.0 ** -11))


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4])
def test_decode_sizes_of_queries(size):
    """The queries' factor into fp16: tiny ones give equal weights, large ones one key."""
    c = Cache([100, 37], 2, 64, 16, 15)
    q = queries(2, 8, 64, 16, size)
    o, tol = attention(c, q, 8, 2.0 ** -11)
    got = decode(c, q, 8).double().view(o.shape)
    assert torch.isfinite(got).all()
    if size < 1:
        assert float(((got - o).abs() - tol).max()) <= 0
    else:  # a weight's error has no bound worth naming; the largest keys lead by far and win
        lead = (got - o).abs().amax() / o.abs().amax()
        assert float(lead) < 2.0 ** -6


def test_decode_values_of_very_different_sizes():
    """Values' scales from 2^-60 to 2^40 in one history: the largest so far is the weights' reference."""
    ctx = [200, 77, 500]
    c = Cache(ctx, 2, 128, 16, 17, amp=lambda x, g: torch.where(torch.arange(2, device=DEV).view(1, 2, 1, 1, 1) == 1, torch.exp2(
        (torch.rand(x.shape[0], 1, 1, x.shape[3], 1, generator=g, device=DEV) * 100 - 60).round()), torch.ones((), device=DEV)))
    q = queries(len(ctx), 16, 128, 18)
    near(decode(c, q, 16), attention(c, q, 16, 2.0 ** -11))


def test_decode_zero_rows_and_rows_without_numbers():
    c = Cache([50, 50, 50], 1, 64, 16, 19)
    zero, bad_k, bad_v = (int(c.table[b, 1]) for b in range(3))
    c.pool[zero, 1, 0, 3], c.scale[zero, 1, 0, 3] = 0, 0.0
    c.value[zero, 1, 0, 3] = 0
    c.scale[bad_k, 0, 0, 2] = NAN
    c.scale[bad_v, 1, 0, 2] = NAN
    q = queries(3, 4, 64, 20)
    out = decode(c, q, 4)
    assert bool(out[1:].isnan().all())
    o, tol = attention(c, q, 4, 2.0 ** -11)
    assert float(((out[0].double().view(4, 64) - o[0]).abs() - tol[0]).max()) <= 0


def test_decode_again_and_on_another_stream_and_from_a_graph():
    ctx = [3000, 10, 777, 0, 64]
    c = Cache(ctx, 4, 128, 64, 21)
    q = queries(len(ctx), 16, 128, 22)
    area, rows, lens = scratch(5, 16, 4, 128), dev_i32(np.arange(5)), dev_i32(ctx)
    first = decode(c, q, 16, area=area)
    near(first, attention(c, q, 16, 2.0 ** -11))
    for _ in range(3):
        assert torch.equal(decode(c, q, 16, area=area), first)
    small = Cache([5], 1, 64, 8, 23)  # another shape in between, on the same scratch
    decode(small, queries(1, 1, 64, 24), 1, area=area)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(decode(c, q, 16, C.c_void_p(side.cuda_stream), area), first)
    out = G.empty((5, 16 * 128), torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        check(lib().dis_k_attn_paged_i8(ptr(q), ptr(c.pool), ptr(c.scale), ptr(c.d_table), c.width, ptr(rows), ptr(lens), ptr(out), ptr(area), 5, 16, 4,
                                        128, 64, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    for _ in range(2):
        out.zero_()
        graph.replay()
        sync()
        assert torch.equal(out, first)


def test_decode_pool_behind_4_gb():
    """Pages whose rows start behind 2^32 bytes."""
    nkv, d, page = 8, 128, 64
    plane = 2 * nkv * page
    n_pages = (1 << 32) // (plane * d) + 40
    pool = torch.empty(n_pages, 2, nkv, page, d, dtype=torch.int8, device=DEV)
    scale = torch.empty(n_pages, 2, nkv, page, device=DEV)
    c = Cache([900, 120], nkv, d, page, 25)
    far = n_pages - 1 - np.arange(c.n_pages)
    pool[torch.from_numpy(far).to(DEV)] = c.pool
    scale[torch.from_numpy(far).to(DEV)] = c.scale
    q = queries(2, 32, d, 26)
    want = attention(c, q, 32, 2.0 ** -11)
    c.pool, c.scale, c.d_table = pool, scale, dev_i32(np.where(c.table < c.n_pages, far[np.minimum(c.table, c.n_pages - 1)], c.table))
    near(decode(c, q, 32), want)
    back = torch.zeros(c.n_pages, 2, nkv, page, d, dtype=torch.bfloat16, device=DEV)
    check(lib().dis_k_kv_read_i8(ptr(pool), ptr(scale), ptr(back), ptr(c.d_table), ptr(dev_i32(c.table)), c.width, ptr(dev_i32([0, 1])), None,
                                 ptr(dev_i32(c.ctx)), 2, nkv, d, page, None))
    sync()
    used = c.used.to(DEV)[:, None, None, :, None].expand(back.shape)
    assert torch.equal(back[used], c.value.float().to(torch.bfloat16)[used])


# ------------------------------------------------------------------------------------------------ writing and reading back
def write(qkv, pool, scale, table, rows, pos, cos, sin, nh, nkv, d, page, stream=None):
    S, T = qkv.shape[0], qkv.shape[1]
    q = G.empty((T, nh * d), torch.bfloat16)
    check(lib().dis_k_rope_kv_write_i8(ptr(qkv), S, T * (nh + 2 * nkv) * d, ptr(q), ptr(pool), ptr(scale), ptr(table), table.shape[1], ptr(rows), ptr(pos),
                                       ptr(cos), ptr(sin), T, nh, nkv, d, page, stream))
    sync()
    return q


def tables(n, d):
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    return guarded(a.cos().float()), guarded(a.sin().float())


def turned(qkv, pos, cos, sin, nh, nkv, d):
    x = qkv.double().sum(0).view(-1, nh + 2 * nkv, d)
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    a, b = x[..., :d // 2], x[..., d // 2:]
    rot = torch.cat([a * c - b * s, b * c + a * s], -1)
    return rot[:, :nh], torch.stack([rot[:, nh:nh + nkv], x[:, nh + nkv:]], 1)  # q [T][nh][d], kv [T][2][nkv][d]


@pytest.mark.parametrize("nh,nkv,d,page,S,lens", [(4, 1, 64, 8, 1, [1]), (8, 8, 128, 16, 3, [1, 5, 20]), (32, 8, 128, 64, 4, [1] * 33),
                                                 (32, 4, 64, 16, 2, [200, 7]), (6, 3, 64, 32, 1, [33, 64, 65]), (64, 8, 128, 128, 8, [3, 130])])
def test_write_and_read(nh, nkv, d, page, S, lens):
    g, past = gen(nh + d), [int(v) for v in np.random.default_rng(3).integers(0, 100, len(lens))]
    total = [a + b for a, b in zip(past, lens)]
    T = sum(lens)
    pages = [-(-t // page) for t in total]
    order = np.random.default_rng(4).permutation(sum(pages) + 2)
    table = np.full((len(lens), max(pages) + 1), 1 << 29, np.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    qkv = guarded(torch.randn(S, T, (nh + 2 * nkv) * d, generator=g, device=DEV))
    rows = dev_i32(np.repeat(np.arange(len(lens)), lens))
    pos = dev_i32(np.concatenate([np.arange(a, a + n) for a, n in zip(past, lens)]))
    cos, sin = tables(max(total), d)
    pool, scale = G.empty((len(order), 2, nkv, page, d), torch.int8), G.empty((len(order), 2, nkv, page))
    before, s_before = pool.clone(), scale.clone()
    d_table = dev_i32(table)
    q = write(qkv, pool, scale, d_table, rows, pos, cos, sin, nh, nkv, d, page)
    want_q, want = turned(qkv, pos, cos, sin, nh, nkv, d)
    size = qkv.double().abs().sum(0).view(T, nh + 2 * nkv, d).amax(-1)  # fp32 sums and products: a few 2^-24 of it
    noise = 2.0 ** -21 * size
    assert bool(((q.double().view(T, nh, d) - want_q).abs() <= 2.0 ** -8 * want_q.abs() + noise[:, :nh, None]).all())
    where, slot = torch.from_numpy(table).to(DEV)[rows.long(), pos.long() // page].long(), pos.long() % page
    x8, s = pool[where, :, :, slot], scale[where, :, :, slot]
    top = want.abs().amax(-1)
    noise = noise[:, nh:].view(T, 2, nkv)
    assert bool(((s.double() * 127 - top).abs() <= 2.0 ** -22 * top + noise).all())
    assert int(x8.abs().amax(-1).min()) == 127 and int(x8.min()) >= -127
    assert bool(((x8.double() * s.double()[..., None] - want).abs() <= (s.double() * (0.5 + 2.0 ** -15) + noise)[..., None]).all())
    touched = torch.zeros(len(order), page, dtype=torch.bool, device=DEV)
    touched[where, slot] = True
    keep = ~touched[:, None, None, :].expand(s_before.shape)
    assert torch.equal(pool[keep], before[keep]) and torch.equal(scale[keep], s_before[keep])
    # read back: the new tokens only, then everything, into pages of another table
    dst = np.full(table.shape, 1 << 29, np.int32)
    dst[table < (1 << 29)] = np.random.default_rng(5).permutation(sum(pages))
    for whole in (False, True):
        first = [0] * len(lens) if whole else past
        back = G.zeros((sum(pages) + 1, 2, nkv, page, d), torch.bfloat16)
        want_back = torch.zeros_like(back)
        for b, t in enumerate(total):
            for p in range(first[b], t):
                row = pool[int(table[b, p // page]), :, :, p % page].float() * scale[int(table[b, p // page]), :, :, p % page][..., None]
                want_back[int(dst[b, p // page]), :, :, p % page] = row.to(torch.bfloat16)
        check(lib().dis_k_kv_read_i8(ptr(pool), ptr(scale), ptr(back), ptr(d_table), ptr(dev_i32(dst)), table.shape[1], ptr(dev_i32(np.arange(len(lens)))),
                                     None if whole else ptr(dev_i32(first)), ptr(dev_i32(total)), len(lens), nkv, d, page, None))
        sync()
        assert torch.equal(back, want_back)


def test_write_rows_of_zeros_tiny_rows_and_rows_without_numbers():
    nh, nkv, d, page = 4, 2, 64, 16
    qkv = torch.randn(1, 6, (nh + 2 * nkv) * d, generator=gen(31), device=DEV)
    v = qkv.view(6, nh + 2 * nkv, d)
    v[0, nh] = 0.0                       # k of token 0, head 0
    v[1, nh + nkv] = 2.0 ** -100         # v of token 1, head 0
    v[2, nh + nkv + 1, 5] = math.inf
    v[3, nh + 1, 7] = NAN
    v[4, nh + nkv] *= 1e36 / float(v[4, nh + nkv].abs().max())
    v[5, 0, 3] = NAN                     # q: only q
    qkv = guarded(qkv)
    cos, sin = tables(8, d)
    pool, scale = G.empty((1, 2, nkv, page, d), torch.int8), G.empty((1, 2, nkv, page))
    q = write(qkv, pool, scale, dev_i32([[0]]), dev_i32([0] * 6), dev_i32(np.arange(6)), cos, sin, nh, nkv, d, page)
    assert float(scale[0, 0, 0, 0]) == 0 and int(pool[0, 0, 0, 0].abs().max()) == 0
    assert float(scale[0, 1, 0, 1]) == 0 and int(pool[0, 1, 0, 1].abs().max()) == 0
    assert math.isnan(float(scale[0, 1, 1, 2])) and math.isnan(float(scale[0, 0, 1, 3]))
    assert abs(float(scale[0, 1, 0, 4]) * 127 / 1e36 - 1) < 1e-6
    assert int(scale[0, :, :, :6].isnan().sum()) == 2
    assert bool(q[5, :d].isnan().any()) and not bool(q[:5].isnan().any()) and not bool(q[5, d:].isnan().any())


def test_written_rows_are_attended_over():
    """The three together: a prompt is written, single tokens follow, each reads what was written."""
    nh, nkv, d, page, n = 8, 2, 128, 16, 45
    qkv = guarded(torch.randn(1, n, (nh + 2 * nkv) * d, generator=gen(33), device=DEV))
    cos, sin = tables(n, d)
    table = np.array([[3, 0, 2, 1]], np.int32)
    c = Cache([n], nkv, d, page, 34)
    c.table, c.d_table, c.width = table, dev_i32(table), 4
    c.pool, c.scale = G.empty((4, 2, nkv, page, d), torch.int8), G.empty((4, 2, nkv, page))
    write(qkv[:, :40].contiguous(), c.pool, c.scale, c.d_table, dev_i32([0] * 40), dev_i32(np.arange(40)), cos, sin, nh, nkv, d, page)
    for t in range(40, n):
        q = write(qkv[:, t:t + 1].contiguous(), c.pool, c.scale, c.d_table, dev_i32([0]), dev_i32([t]), cos, sin, nh, nkv, d, page)
        c.ctx = [t + 1]
        out = decode(c, q, nh)
        c.value = c.pool.double() * c.scale.double()[..., None]
        near(out, attention(c, q, nh, 2.0 ** -11))


# ------------------------------------------------------------------------------------------------ shared prefix
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("d,group,nkv,page", [(128, 4, 2, 64), (128, 8, 1, 16), (64, 8, 2, 32), (64, 4, 1, 8), (128, 1, 3, 64), (64, 2, 2, 16)])
@pytest.mark.parametrize("prefix", [0, 1, 100, 640, 1500])
def test_shared_prefix(int8, d, group, nkv, page, prefix):
    own = [1, 0, 17, 300, 64, 5, 128]
    ctx = [prefix + n for n in own]
    c = Cache(ctx, nkv, d, page, prefix + d + group, int8, prefix)
    q = queries(len(ctx), nkv * group, d, prefix)
    near(shared(c, q, nkv * group, prefix), attention(c, q, nkv * group, 2.0 ** -8))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T,group,d", [(1, 4, 128), (33, 4, 128), (64, 8, 128), (130, 1, 64), (70, 8, 64), (16, 8, 128)])
def test_shared_prefix_batches(int8, T, group, d):
    """Batches whose rows fill a product's 128, or do not, or go past them."""
    r = np.random.default_rng(T)
    ctx = [900 + int(v) for v in r.integers(1, 80, T)]
    c = Cache(ctx, 2, d, 64, T, int8, 900)
    q = queries(T, 2 * group, d, T)
    near(shared(c, q, 2 * group, 900), attention(c, q, 2 * group, 2.0 ** -8))


@pytest.mark.parametrize("int8", [False, True])
def test_shared_prefix_with_shorter_histories(int8):
    """Tokens that see a part of the prefix, or nothing, beside tokens that see all of it."""
    ctx = [700, 512, 513, 511, 300, 1, 0, 65, 600]
    c = Cache(ctx, 2, 128, 64, 41, int8, 512)
    q = queries(len(ctx), 8, 128, 42)
    out = shared(c, q, 8, 512)
    near(out, attention(c, q, 8, 2.0 ** -8))
    assert int((out[6] != 0).sum()) == 0


@pytest.mark.parametrize("int8", [False, True])
def test_shared_prefix_long_and_again(int8):
    ctx = [20000 + 37 * t for t in range(24)]
    c = Cache(ctx, 2, 128, 64, 43, int8, 20000)
    q = queries(len(ctx), 8, 128, 44)
    area = scratch(24, 8, 2, 128, True)
    first = shared(c, q, 8, 20000, area=area)
    near(first, attention(c, q, 8, 2.0 ** -8))
    assert torch.equal(shared(c, q, 8, 20000, area=area), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(shared(c, q, 8, 20000, C.c_void_p(side.cuda_stream), area), first)
    out, rows, lens = G.empty((24, 8 * 128), torch.bfloat16), dev_i32(np.arange(24)), dev_i32(ctx)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        check(lib().dis_k_attn_shared(ptr(q), ptr(c.pool), ptr(c.scale), c.n_pages, ptr(c.d_table), c.width, ptr(rows), ptr(lens), 20000, ptr(out), ptr(area),
                                      24, 8, 2, 128, 64, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    for _ in range(2):
        out.zero_()
        graph.replay()
        sync()
        assert torch.equal(out, first)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T,group,d,prefix", [(64, 8, 128, 8000), (40, 4, 128, 5000), (64, 8, 64, 8000), (30, 4, 64, 9000)])
def test_shared_prefix_many_steps_again(int8, T, group, d, prefix):
    """Slices of many key tiles: every run has the same bits, whatever the scratch held."""
    ctx = [prefix + 1 + 7 * t % 300 for t in range(T)]
    c = Cache(ctx, 8, d, 64, T, int8, prefix)
    q = queries(T, 8 * group, d, 5)
    area = scratch(T, 8 * group, 8, d, True)
    first = shared(c, q, 8 * group, prefix, area=area)
    near(first, attention(c, q, 8 * group, 2.0 ** -8))
    for k in range(10):
        area[1 << 16:].fill_(float(k))
        assert torch.equal(shared(c, q, 8 * group, prefix, area=area), first), k


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T,group,nkv,d,page,prefix", [(72, 1, 8, 128, 16, 577), (64, 2, 8, 128, 8, 641), (40, 4, 8, 128, 64, 1250), (57, 8, 8, 128, 32, 896), (33, 4, 8, 128, 128, 1500),
                                                      (80, 8, 8, 64, 8, 1001), (130, 1, 8, 64, 64, 640), (12, 4, 8, 128, 64, 4095), (6, 8, 8, 128, 16, 7000), (9, 2, 16, 64, 64, 5000)])
def test_shared_prefix_read_once(int8, T, group, nkv, d, page, prefix):
    """Sizes at which the prefix is read once: prefixes that end inside a tile and inside a page, one tile of rows and several, rows behind the last, and
    among the histories some that end at the prefix's end, inside it, or are empty."""
    assert lib().dis_k_attn_shared_in_common(T, nkv * group, nkv, d, prefix, int8) == 1
    own = np.random.default_rng(T).integers(0, 90, T)
    ctx = [prefix + int(n) for n in own]
    ctx[1], ctx[2], ctx[3] = prefix, prefix - 1, 0
    ctx[T - 1] = prefix // 2
    c = Cache(ctx, nkv, d, page, T + prefix, int8, prefix)
    q = queries(T, nkv * group, d, prefix)
    area = scratch(T, nkv * group, nkv, d, True)
    out = shared(c, q, nkv * group, prefix, area=area)
    near(out, attention(c, q, nkv * group, 2.0 ** -8))
    assert int((out[3] != 0).sum()) == 0
    area[1 << 16:].fill_(7.0)
    assert torch.equal(shared(c, q, nkv * group, prefix, area=area), out)


def test_shared_prefix_read_once_rows_without_numbers_and_sizes():
    """A NaN among the prefix's keys reaches every token that sees it, in its kv head; scales from 2^-60 to 2^40; large scores."""
    T, prefix = 40, 1250
    ctx = [prefix + 1 + t for t in range(T)]
    ctx[7] = 90
    spread = lambda x, g: torch.where(torch.arange(2, device=DEV).view(1, 2, 1, 1, 1) == 1, torch.exp2(  # noqa: E731
        (torch.rand(x.shape[0], 1, 1, x.shape[3], 1, generator=g, device=DEV) * 100 - 60).round()), torch.ones((), device=DEV))
    c = Cache(ctx, 8, 128, 64, 51, True, prefix, amp=spread)
    for size in (1.5, 30.0, 1e-30):
        q = queries(T, 32, 128, 52, size)
        near(shared(c, q, 32, prefix), attention(c, q, 32, 2.0 ** -8))
    for int8 in (False, True):
        c = Cache(ctx, 8, 128, 64, 53, int8, prefix)
        q = queries(T, 32, 128, 54)
        page = int(c.table[0, 5])  # positions 320 ..
        if int8:
            c.scale[page, 0, 1, 5] = NAN
        else:
            c.pool[page, 0, 1, 5] = NAN
        out = shared(c, q, 32, prefix).view(T, 32, 128)
        seen = [t for t in range(T) if t != 7]
        assert bool(out[seen][:, 4:8].isnan().all())
        o, tol = attention(c, q, 32, 2.0 ** -8)
        ok = (out.double() - o).abs() <= tol
        assert bool(ok[:, :4].all()) and bool(ok[:, 8:].all()) and bool(ok[7].all())


def test_shared_prefix_sizes():
    """Large scores (one key wins), and values' scales from 2^-60 to 2^40, in 8-bit pages."""
    ctx = [700 + t for t in range(20)]
    c = Cache(ctx, 2, 128, 64, 45, True, 640, amp=lambda x, g: torch.where(torch.arange(2, device=DEV).view(1, 2, 1, 1, 1) == 1, torch.exp2(
        (torch.rand(x.shape[0], 1, 1, x.shape[3], 1, generator=g, device=DEV) * 100 - 60).round()), torch.ones((), device=DEV)))
    q = queries(len(ctx), 16, 128, 46)
    near(shared(c, q, 16, 640), attention(c, q, 16, 2.0 ** -8))
    q = queries(len(ctx), 16, 128, 47, 30.0)
    near(shared(c, q, 16, 640), attention(c, q, 16, 2.0 ** -8))


@pytest.mark.parametrize("int8", [False, True])
def test_shared_prefix_row_without_numbers(int8):
    """A NaN in one kv head of the prefix reaches that head's results of all tokens that see it, and no others."""
    ctx = [300, 320, 90, 301]
    c = Cache(ctx, 2, 128, 64, 48, int8, 256)
    q = queries(4, 8, 128, 49)
    page = int(c.table[0, 2])  # positions 128 ..
    if int8:
        c.scale[page, 0, 1, 5] = NAN
    else:
        c.pool[page, 0, 1, 5] = NAN
    out = shared(c, q, 8, 256).view(4, 8, 128)
    assert bool(out[[0, 1, 3]][:, 4:].isnan().all())
    o, tol = attention(c, q, 8, 2.0 ** -8)
    ok = (out.double() - o).abs() <= tol
    assert bool(ok[:, :4].all()) and bool(ok[2].all())


# ------------------------------------------------------------------------------------------------ refusals
def refused(rc, word):
    assert rc == B.ERR_INVALID_ARGUMENT
    assert word in lib().dis_last_error().decode()


def test_refusals():
    t = G.zeros(1 << 16)
    p, odd = ptr(t), C.c_void_p(t.data_ptr() + 2)
    W = lambda **k: lib().dis_k_rope_kv_write_i8(*dict(dict(qkv=p, n=1, st=0, q=p, pool=p, scale=p, pt=p, mp=4, row=p, pos=p, c=p, s=p, T=1, nh=4, nkv=2,  # noqa: E731
                                                            d=64, page=16, stream=None), **k).values())
    R = lambda **k: lib().dis_k_kv_read_i8(*dict(dict(pool=p, scale=p, kv=p, src=p, dst=p, mp=4, row=p, first=None, ctx=p, n=1, nkv=2, d=64, page=16,  # noqa: E731
                                                      stream=None), **k).values())
    A = lambda **k: lib().dis_k_attn_paged_i8(*dict(dict(q=p, pool=p, scale=p, pt=p, mp=4, row=p, ctx=p, out=p, area=p, T=1, nh=4, nkv=2, d=64, page=16,  # noqa: E731
                                                         stream=None), **k).values())
    S = lambda **k: lib().dis_k_attn_shared(*dict(dict(q=p, pool=p, scale=None, np=4, pt=p, mp=4, row=p, ctx=p, prefix=16, out=p, area=p, T=1, nh=4, nkv=2,  # noqa: E731
                                                       d=64, page=16, stream=None), **k).values())
    for f in (W, A, S):
        refused(f(T=-1), "negative")
        refused(f(nh=6), "n_heads")
        refused(f(nh=5), "n_heads")
        refused(f(nkv=0), "n_heads")
        assert f(T=0) == B.OK
    for f in (W, R, A, S):
        refused(f(d=96), "head_dim")
        refused(f(page=12), "page_size")
        refused(f(page=4), "page_size")
        refused(f(mp=0), "max_pages")
        refused(f(mp=1 << 28), "max_pages")
    for f, names in ((W, ["qkv", "q", "pool", "scale", "pt", "row", "pos", "c", "s"]), (R, ["pool", "scale", "kv", "src", "dst", "row", "ctx"]),
                     (A, ["q", "pool", "scale", "pt", "row", "ctx", "out", "area"]), (S, ["q", "pool", "pt", "row", "ctx", "out", "area"])):
        for n in names:
            refused(f(**{n: None}), "null")
    for f, names in ((W, ["qkv", "c", "s", "q", "pool"]), (R, ["pool", "kv"]), (A, ["q", "pool", "area", "out"]), (S, ["q", "pool", "area", "out"])):
        for n in names:
            refused(f(**{n: odd}), "start")
    refused(W(n=0), "n_partial")
    refused(W(n=2, st=6), "start")
    assert R(n=0) == B.OK
    refused(R(n=-1), "negative")
    refused(R(mp=70000), "65535")
    refused(S(prefix=-1), "prefix")
    refused(S(prefix=65), "prefix")
    refused(S(np=0), "n_pages")
    refused(S(np=1 << 40), "n_pages")
    sync()
