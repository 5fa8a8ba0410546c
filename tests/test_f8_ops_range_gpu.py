"""Products in 8-bit floating point whose two scales together leave the range of fp32 (weights' scales are any fp32 number): zeros stay zeros and numbers
numbers where the product of the scales is too large to be one, and where it is too small to be held in full a block is off by up to 2^-125 more (half a step
of the smallest numbers, 2^-150, times a sum of at most 2^25).  Gate-up products of few tokens hold sums with a product that is too large in units of 2^24,
and the half step is one of units there: 2^-150 2^25 2^24 = 2^-101.  The other bounds as in test_f8_ops_gpu.py."""
import pytest
import torch

from distributed_inference_server_b200 import binding as B
from tests import _gpu_util as G
from tests._gpu_util import DEV, check, lib, ptr, sync
from tests.test_f8_ops_gpu import F8, blocks, gen, guarded, near_8_bits, product, silu64, sums_off

pytestmark = pytest.mark.gpu
LEAST, LARGE = 0x01, 0x7c  # 2^-9 and 384 in e4m3


def values(q, s, weight):
    """What 8-bit rows [T][K] under [blocks][T], or a weight [N][K] under [blocks][blocks], stand for, in 64 bits"""
    s = (s.repeat_interleave(128, 0)[:q.shape[0]] if weight else s.T).double()
    return q.view(F8).double() * s.repeat_interleave(128, 1)[:, :q.shape[1]]


def some(g, n, k):
    """e4m3 numbers around 1, both signs"""
    return (torch.randn(n, k, generator=g, device=DEV).clamp(-4, 4)).to(F8).view(torch.uint8)


def wild_rows(g, T, K):
    """Tokens of three kinds: ordinary ones (blocks 0 and 4), ones with a block whose scales vanish together (2), ones with a block whose scales are too large
    together (3).  Block 1 is zero, under a scale that is too large with the weight's."""
    x8, xs = torch.zeros(T, K, dtype=torch.uint8, device=DEV), torch.ones(blocks(K), T, device=DEV)
    kind = torch.arange(T, device=DEV) % 3
    fill = lambda v: torch.tensor(v, dtype=torch.uint8, device=DEV)  # noqa: E731
    for b in (0, 4):
        x8[:, b * 128:(b + 1) * 128] = torch.where((kind == 0)[:, None], some(g, T, K)[:, b * 128:(b + 1) * 128], fill(0))
    x8[:, 256:384] = torch.where((kind == 1)[:, None], fill(LARGE), fill(0))
    x8[:, 384:512] = torch.where((kind == 2)[:, None], fill(LEAST), fill(0))
    xs[0], xs[1], xs[2], xs[3], xs[4] = 0.25, 2.0 ** 100, 2.0 ** -80, 2.0 ** 70, 2.0 ** 100
    return x8, xs, kind


def wild_weight(g, N, K, small, large):
    """The weight that goes with them: scales per block of K, the same for all rows but for a factor; a zero scale for block 4's second half of the rows"""
    w8 = some(g, N, K)
    w8[:, 256:384], w8[:, 384:512] = LARGE, LEAST
    ws = torch.empty(blocks(N), blocks(K), device=DEV)
    f = 1 + torch.rand(blocks(N), generator=g, device=DEV) / 4
    ws[:, 0], ws[:, 1], ws[:, 2], ws[:, 3], ws[:, 4] = 0.01 * f, 2.0 ** 60 * f, small * f, large * f, 2.0 ** -104 * f
    ws[blocks(N) // 2:, 4] = 0
    ws[:, 5:] = 1.0
    return w8, ws


def off(xv, wv, least=2.0 ** -125):
    return sums_off(xv, wv) + blocks(xv.shape[1]) * least


# in tiles with and without slices of K, in pairs of 128 and of 256 columns
@pytest.mark.parametrize("T,N,K", [(3, 400, 656), (100, 1001, 640), (40, 20000, 640), (300, 400, 656), (400, 300, 640), (1300, 8192, 640), (1300, 8200, 656)])
@pytest.mark.parametrize("bf16", [False, True])
def test_scales_that_leave_the_range_together(T, N, K, bf16):
    g = gen(T + N)
    x8, xs, kind = wild_rows(g, T, K)
    w8, ws = wild_weight(g, N, K, 1.37 * 2.0 ** -55, -1.2 * 2.0 ** 62)  # 2^-135 and 2^132 with the rows'
    out = product(guarded(x8), guarded(xs), guarded(w8), guarded(ws), T, N, K, bf16)
    sync()
    xv, wv = values(x8, xs, False), values(w8, ws, True)
    want, bound = xv @ wv.T, off(xv, wv)
    if bf16:
        bound = bound + (want.abs() + bound) * 2.0 ** -8
    assert float(want[kind == 1].abs().min()) > 2.0 ** -112 and float(want[kind == 2].abs().max()) > 2.0 ** 118
    assert bool(((out.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("T,N,K", [(3, 400, 656), (100, 1001, 640), (300, 400, 656), (1300, 8192, 640)])
def test_scales_that_vanish_together(T, N, K):
    """Without any that are too large: down to the smallest numbers, and zeros under whatever scale."""
    g = gen(T + N)
    x8, xs, kind = wild_rows(g, T, K)
    xs[1], xs[3] = 2.0 ** -126, 2.0 ** -126  # (as zeros have it; kind 2: the smallest values there are)
    w8, ws = wild_weight(g, N, K, 1.37 * 2.0 ** -55, 2.0 ** -5)
    out = product(guarded(x8), guarded(xs), guarded(w8), guarded(ws), T, N, K)
    sync()
    xv, wv = values(x8, xs, False), values(w8, ws, True)
    want, bound = xv @ wv.T, off(xv, wv)
    assert float(want[kind == 1].abs().min()) > 2.0 ** -112 and 0 < float(want[kind == 2].abs().max()) < 2.0 ** -140
    assert bool(((out.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("T,N,K", [(3, 400, 656), (100, 1001, 640), (40, 20000, 640), (400, 300, 640), (700, 400, 656), (1300, 8192, 640), (6000, 1030, 656)])
def test_one_wild_token_among_ordinary_ones(T, N, K):
    """A few tokens whose zeros stand under a scale that is too large, here and there: they are what they would be, and so are the others."""
    g = gen(T + N)
    x8, xs, w8 = some(g, T, K), torch.rand(blocks(K), T, generator=g, device=DEV) + 0.5, some(g, N, K)
    ws = torch.rand(blocks(N), blocks(K), generator=g, device=DEV) + 0.5
    xs[1] *= 2.0 ** -40
    ws[:, 1] *= 2.0 ** 40
    wild = torch.arange(T // 2, T, 129, device=DEV)
    x8[wild, 128:256] = 0
    xs[1, wild] = 2.0 ** 100
    out = product(guarded(x8), guarded(xs), guarded(w8), guarded(ws), T, N, K)
    sync()
    xv, wv = values(x8, xs, False), values(w8, ws, True)
    assert bool(((out.double() - xv @ wv.T).abs() <= off(xv, wv)).all())


@pytest.mark.parametrize("T,I,K", [(3, 400, 656), (100, 720, 640), (17, 16384, 640), (300, 400, 656), (700, 1040, 640)])
def test_gate_up_scales_that_leave_the_range_together(T, I, K):
    g = gen(T + I)
    x8, xs, _ = wild_rows(g, T, K)
    gq, gs = wild_weight(g, I, K, 2.0 ** 57, 2.0 ** -70)            # gates of ordinary size ...
    uq, us = wild_weight(g, I, K, 1.37 * 2.0 ** -55, 1.2 * 2.0 ** 62)  # ... and up of 2^-135 and 2^132 times the block's sum
    h8, hs = G.empty((T, I), torch.uint8), G.empty((blocks(I), T))
    check(lib().dis_k_gemm_silu_f8(ptr(guarded(x8)), ptr(guarded(xs)), ptr(guarded(torch.cat([gq, uq]))), ptr(guarded(torch.cat([gs, us]))), ptr(h8), ptr(hs), T, I, K, None))
    sync()
    xv, gv, uv = values(x8, xs, False), values(gq, gs, True), values(uq, us, True)
    a, b, oa, ob = xv @ gv.T, xv @ uv.T, off(xv, gv, 2.0 ** -101), off(xv, uv, 2.0 ** -101)
    want = silu64(a) * b
    near_8_bits(h8, hs, want, 1.1 * oa * (b.abs() + ob) + silu64(a).abs() * ob + want.abs() * 2.0 ** -17)


@pytest.mark.parametrize("T,N,K", [(40, 400, 656), (300, 400, 656), (1300, 8192, 640)])
def test_what_is_no_number_stays_none(T, N, K):
    """Among wild scales: a result beyond fp32 is infinite, and an infinite or NaN scale makes of its token's row or its weight's columns what the definition
    makes of them, and leaves the rest as it is."""
    g = gen(T)
    x8, xs, kind = wild_rows(g, T, K)
    w8, ws = wild_weight(g, N, K, 1.37 * 2.0 ** -55, 1.2 * 2.0 ** 62)
    ws[0, 3] = 2.0 ** 90  # 2^160 with the rows', 2^149 times the least of sums
    clean = product(guarded(x8), guarded(xs), guarded(w8), guarded(ws), T, N, K)
    sync()
    assert bool((clean[kind == 2, :128] == float("inf")).all()) and bool(clean[kind != 2].isfinite().all()) and bool(clean[:, 128:].isfinite().all())
    ws[1, 2] = float("inf")    # times the sums of kind 1 an infinity, times the others' zeros NaN
    xs[3, 5] = float("nan")
    out = product(guarded(x8), guarded(xs), guarded(w8), guarded(ws), T, N, K)
    sync()
    lost = torch.zeros(T, N, dtype=torch.bool, device=DEV)
    lost[kind != 1, 128:256] = True
    lost[5] = True
    assert torch.equal(out.isnan(), lost)
    assert bool((out[kind == 1, 128:256] == float("inf")).all())
    rest = ~lost
    rest[kind == 1, 128:256] = False
    assert torch.equal(out[rest], clean[rest])


def test_wild_tokens_among_many_tiles():
    """More than 256 tiles a CTA, which note what they have to look at again in 256 bits; captured, and replayed with other tokens."""
    T, N, K = 40000, 32000, 16
    g = gen(7)
    x8, w8 = some(g, T, K), some(g, N, K)
    xs = (torch.rand(1, T, generator=g, device=DEV) + 0.5) * 2.0 ** -60
    ws = (torch.rand(blocks(N), 1, generator=g, device=DEV) + 0.5) * 2.0 ** 60
    out = torch.empty(T, N, dtype=torch.bfloat16, device=DEV)
    x, s = x8.clone(), xs.clone()

    def call(stream):
        check(lib().dis_k_gemm_f8(ptr(x), ptr(s), ptr(w8), ptr(ws), ptr(out), B.BF16, T, N, K, stream.cuda_stream))

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    call(st)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        call(torch.cuda.current_stream())
    for wild in ((5, T - 1), (), (0, 255, 256, 20001)):
        x.copy_(x8)
        s.copy_(xs)
        out.fill_(float("nan"))
        for t in wild:
            x[t], s[0, t] = 0, 2.0 ** 100
        graph.replay()
        sync()
        assert bool(out.isfinite().all())
        for t in (0, 5, 128, 256, 20001, T - 1):
            xv, wv = values(x[t:t + 1], s[:, t:t + 1], False), values(w8, ws, True)
            want, bound = xv @ wv.T, off(xv, wv)
            bound = bound + (want.abs() + bound) * 2.0 ** -8
            assert bool(((out[t:t + 1].double() - want).abs() <= bound).all()), t
