"""Products in 8-bit floating point (rows and weights turned into 8 bits, the residual add and norm in front, plain and gate-up products, a whole feed-forward
block) through the C ABI, against the definitions in 64 bits.  Every bound follows from the roundings that the operators make:
  8-bit values   bit for bit where the input is given: x / s is exact for a power of two s, and e4m3 rounds to nearest, ties to even;
  e4m3           half a step: 2^-4 of the value, 2^-10 of the scale below 2^-6 of it;
  a block's sum  128 products (exact in fp32), added with an error of at most one part in 2^23 of what has been added so far each: 2^-16 sum |x w|;
  blocks         each block's sum times its two scales, added in fp32: 2^-23 per block (a product of scales, an FMA);
  bf16           half a step is at most 2^-8 of the result.
"""
import numpy as np
import pytest
import torch

from distributed_inference_server_b200 import binding as B
from tests import _gpu_util as G
from tests._gpu_util import DEV, check, lib, ptr, sync

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def guarded(t):
    x = G.empty(t.shape, t.dtype)
    x.copy_(t)
    return x


def blocks(n):
    return -(-n // 128)


def padded(x, rows, cols):
    return torch.nn.functional.pad(x, (0, cols - x.shape[1], 0, rows - x.shape[0]))


def scales_of(top):
    """2^ceil(log2(top / 448)), not below 2^-126, NaN where top is not finite; top in fp64"""
    m, e = torch.frexp(top / 448)  # (1 / 448 is no power of two: exact ties of the division only where it is exact)
    s = torch.where(top > 0, torch.ldexp(torch.ones_like(m), e - (m == 0.5).int()), 0.0).clamp_min(2.0 ** -126)  # (a block of zeros has the smallest)
    return torch.where(torch.isfinite(top), s, float("nan"))


def rows_in_8_bits(x):
    """x [T][K] in fp64 -> (e4m3 bytes [T][K], scales [ceil(K / 128)][T], values in fp64)"""
    T, K = x.shape
    b = padded(x, T, blocks(K) * 128).view(T, -1, 128)
    s = scales_of(torch.where(b.isnan(), float("inf"), b.abs()).amax(-1))
    q = (b / s[..., None]).float().to(F8)
    return q.view(T, -1)[:, :K].contiguous(), s.T.contiguous().float(), (q.double() * s[..., None]).view(T, -1)[:, :K]


def weight(g, n, k, pow2=False):
    """(e4m3 [n][k], scales [ceil(n / 128)][ceil(k / 128)], values in fp64)"""
    w = padded(torch.randn(n, k, generator=g, device=DEV, dtype=torch.float64) * k ** -0.5, blocks(n) * 128, blocks(k) * 128)
    b = w.view(blocks(n), 128, blocks(k), 128)
    top = b.abs().amax((1, 3))
    s = scales_of(top) if pow2 else (top / 448).float().double()
    q = (b / s[:, None, :, None]).clamp(-448, 448).float().to(F8)
    return q.view(blocks(n) * 128, -1)[:n, :k].contiguous(), s.float(), (q.double() * s[:, None, :, None]).view(blocks(n) * 128, -1)[:n, :k]


def rows(g, t, k):
    x = torch.randn(t, k, generator=g, device=DEV) * (torch.rand(t, 1, generator=g, device=DEV) * 2 + 0.3) * (torch.rand(k, generator=g, device=DEV) + 0.5)
    x[:, torch.randint(0, k, (max(1, k // 100),), generator=g, device=DEV)] *= 15
    return x.to(torch.bfloat16)


def same_bits(a, b):
    """Equal bytes; any NaN equals any NaN."""
    a, b = a.view(torch.uint8), b.view(torch.uint8)
    return bool(((a == b) | (((a & 0x7f) == 0x7f) & ((b & 0x7f) == 0x7f))).all())


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


# ------------------------------------------------------------------------------------------------ into 8 bits
def quant(x):
    T, K = x.shape
    x8, s = G.empty((T, K), torch.uint8), G.empty((blocks(K), T))
    check(lib().dis_k_quant_f8(ptr(x), ptr(x8), ptr(s), T, K, None))
    sync()
    return x8, s


@pytest.mark.parametrize("T,K", [(1, 16), (1, 4096), (3, 128), (16, 144), (17, 1040), (33, 2048), (300, 272), (1, 14336), (2049, 512)])
def test_rows_into_8_bits(T, K):
    g = gen(T * 7 + K)
    x = rows(g, T, K)
    x[0, 0] = 448.0
    if T > 2:
        x[1] = 0
        x[2, :16] = torch.tensor([1.0, 1.0625, 1.1875, -1.0625, 448, 447, 432, 416, 0.0156, 0.001, 0.0009765, -0.0029, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 0], device=DEV)
        x[2, 16:] = 0
    q, s, _ = rows_in_8_bits(x.double())
    x8, xs = quant(guarded(x))
    assert torch.equal(xs, s)
    assert same_bits(x8, q)


def test_rows_at_the_ends_of_the_range():
    """The largest and smallest bf16 numbers, maxima at and beside 448 times a power of two, infinities and NaN: only their own block is lost."""
    tops = [448.0, 450.0, 446.0, 3.38953139e38, 2.0 ** -120, 1.75 * 2.0 ** -126, 2.0 ** -133, 7.0 * 2.0 ** -20, 7.03125 * 2.0 ** -20, 0.0, float("inf"), -float("inf"), float("nan")]
    x = torch.randn(len(tops), 256, generator=gen(5), device=DEV).clamp(-4, 4) / 4
    for i, t in enumerate(tops):
        x[i, :128] *= min(abs(t), 3e38) if t == t else 1.0
        x[i, 77] = t
    x = x.to(torch.bfloat16)
    q, s, _ = rows_in_8_bits(x.double())
    x8, xs = quant(guarded(x))
    assert same(xs, s)
    assert xs[0, 9] == 2.0 ** -126 and xs[0, 10:].isnan().all() and xs[1].isfinite().all()
    fine = torch.cat([s[0].isfinite()[:, None].expand(-1, 128), torch.ones(len(tops), 128, dtype=torch.bool, device=DEV)], 1)
    assert same_bits(x8.view(torch.uint8)[fine], q.view(torch.uint8)[fine])


@pytest.mark.parametrize("N,K", [(1, 16), (128, 128), (129, 144), (1000, 1040), (4096, 512)])
def test_weights_into_8_bits(N, K):
    g = gen(N + K)
    w = (torch.randn(N, K, generator=g, device=DEV) * torch.rand(K, generator=g, device=DEV)).to(torch.bfloat16)
    if N > 128:
        w[128:, :] = 0
    b = padded(w.double(), blocks(N) * 128, blocks(K) * 128).view(blocks(N), 128, blocks(K), 128)
    s = scales_of(b.abs().amax((1, 3)))
    q = (b / s[:, None, :, None]).float().to(F8).view(blocks(N) * 128, -1)[:N, :K].contiguous()
    w8, ws = G.empty((N, K), torch.uint8), G.empty((blocks(N), blocks(K)))
    check(lib().dis_k_quant_weight_f8(ptr(guarded(w)), ptr(w8), ptr(ws), N, K, None))
    sync()
    assert torch.equal(ws, s.float())
    assert same_bits(w8, q)


def near_8_bits(x8, s, want, off):
    """Values held in 8 bits against what was rounded, itself known to `off` (absolute): half a step of e4m3 more; the scale that of the maximum, give or take off."""
    K = want.shape[1]
    S = s.double().T.repeat_interleave(128, 1)[:, :K]
    got = x8.view(F8).double() * S
    bound = torch.maximum((want.abs() + off) * 2.0 ** -4, S * 2.0 ** -10) + off
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() - bound).max())
    T = want.shape[0]
    pad = lambda v: padded(v, T, blocks(K) * 128).view(T, -1, 128).amax(-1)  # noqa: E731
    lo, hi = scales_of((pad(want.abs()) - pad(off)).clamp_min(0)), scales_of(pad(want.abs()) + pad(off))
    assert bool(((s.T.double() >= lo) & (s.T.double() <= hi)).all())


@pytest.mark.parametrize("T,H,n_partial,how", [(1, 4096, 4, "add"), (32, 4096, 1, "add"), (5, 272, 3, "add"), (700, 2048, 2, "add"), (3, 8192, 8, "add"), (2, 16, 1, "add"),
                                               (40, 4096, 0, "embed"), (2, 51200, 1, "add"), (513, 20000, 1, "add"), (513, 6160, 2, "add"), (513, 12288, 1, "embed"), (1, 12288, 3, "add"), (600, 272, 0, "embed"), (7, 1040, 2, "map"), (520, 8192, 0, "map")])
def test_norm_into_8_bits(T, H, n_partial, how):
    g = gen(T + H)
    rows_in = 2 * T if how == "map" else T
    x0 = torch.randn(rows_in, H, generator=g, device=DEV) * 3
    part = torch.randn(max(n_partial, 1), rows_in, H, generator=g, device=DEV)
    gain = 1 + 0.2 * torch.randn(H, generator=g, device=DEV)
    embed = (torch.randn(50, H, generator=g, device=DEV)).to(torch.bfloat16)
    ids = torch.randint(0, 50, (T,), generator=g, device=DEV, dtype=torch.int32)
    rmap = torch.randperm(rows_in, generator=g, device=DEV)[:T].int()
    x = guarded(x0)
    x8, s = G.empty((T, H), torch.uint8), G.empty((blocks(H), T))
    check(lib().dis_k_add_rmsnorm_f8(ptr(x), ptr(guarded(ids)) if how == "embed" else None, ptr(guarded(embed)) if how == "embed" else None, ptr(guarded(part)), n_partial,
                                     rows_in * H, ptr(guarded(gain)), ptr(x8), ptr(s), ptr(guarded(rmap)) if how == "map" else None, T, H, 1e-5, None))
    sync()
    want = embed.double()[ids.long()] if how == "embed" else x0.double() + part[:n_partial].double().sum(0)
    mag = want.abs() if how == "embed" else x0.double().abs() + part[:n_partial].double().abs().sum(0)
    if how == "map":
        assert torch.equal(x, x0)
        want, mag = want[rmap.long()], mag[rmap.long()]
    else:
        assert bool(((x.double() - want).abs() <= n_partial * 2.0 ** -24 * mag).all())
    n = want / (want.square().mean(-1, keepdim=True) + 1e-5).sqrt() * gain.double()
    # the row's own roundings, the mean's (sums of at most 13 terms in a thread, then trees: 2^-19) and the reciprocal root's (2^-22)
    off = n.abs() * 2.0 ** -18 + mag * n_partial * 2.0 ** -24 * (n.abs() / want.abs().clamp_min(1e-300)).clamp_max(1e30)
    near_8_bits(x8, s, n, off)


# ------------------------------------------------------------------------------------------------ products
def product(xq, xs, wq, ws, T, N, K, bf16=False):
    out = G.empty((T, N), torch.bfloat16 if bf16 else torch.float32)
    check(lib().dis_k_gemm_f8(ptr(xq), ptr(xs), ptr(wq), ptr(ws), ptr(out), B.BF16 if bf16 else B.F32, T, N, K, None))
    return out


def sums_off(xv, wv):
    return (2.0 ** -16 + blocks(xv.shape[1]) * 2.0 ** -23) * (xv.abs() @ wv.abs().T)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,N,K", [(1, 4096, 4096), (1, 1, 16), (2, 130, 272), (31, 1001, 1040), (32, 6144, 4096), (33, 256, 128), (64, 512, 2048), (65, 2560, 2048),
                                   (77, 1001, 1040), (128, 128, 14336), (129, 300, 400), (256, 4096, 1024), (257, 512, 512), (300, 1001, 1040), (513, 260, 144),
                                   (1000, 2048, 5632), (2100, 4096, 256), (2100, 5001, 656), (1300, 8200, 1040), (3000, 4096, 1936), (1, 20000, 128), (5, 128, 28672), (700, 8, 16)])
def test_product(T, N, K, bf16):
    g = gen(T + 3 * N + K)
    xq, xs, xv = rows_in_8_bits(rows(g, T, K).double())
    wq, ws, wv = weight(g, N, K)
    out = product(guarded(xq.view(torch.uint8)), guarded(xs), guarded(wq.view(torch.uint8)), guarded(ws), T, N, K, bf16)
    sync()
    want, bound = xv @ wv.T, sums_off(xv, wv)
    if bf16:
        bound = bound + (want.abs() + bound) * 2.0 ** -8
    assert bool(((out.double() - want).abs() <= bound).all()), float(((out.double() - want).abs() / bound.clamp_min(1e-300)).max())


@pytest.mark.parametrize("T", [3, 100, 400])
def test_lost_blocks_stay_where_they_are(T):
    """A NaN scale of one token's block loses that token's row, one of the weight's its 128 columns, NaN values in the rows likewise; the rest is what it was.  Wild scales
    (zeros, very large and small ones, negative ones) are numbers like others."""
    g, N, K = gen(T), 400, 656
    xq, xs, xv = rows_in_8_bits(rows(g, T, K).double())
    wq, ws, wv = weight(g, N, K)
    ws[0, 0], ws[0, 1], ws[0, 2], ws[0, 3] = 0.0, -3.0, 1e20, 1e-30
    s = ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    wv = wq.double() * s
    clean = product(guarded(xq.view(torch.uint8)), guarded(xs), guarded(wq.view(torch.uint8)), guarded(ws), T, N, K)
    sync()
    assert bool(((clean.double() - xv @ wv.T).abs() <= sums_off(xv, wv)).all())
    xs[2, T // 2] = float("nan")
    ws[2, 5] = float("nan")
    w8 = wq.view(torch.uint8).clone()
    w8[399, 3] = 0x7f
    out = product(guarded(xq.view(torch.uint8)), guarded(xs), guarded(w8), guarded(ws), T, N, K)
    sync()
    lost = torch.zeros(T, N, dtype=torch.bool, device=DEV)
    lost[T // 2] = True
    lost[:, 256:384] = True
    lost[:, 399] = True
    assert torch.equal(out.isnan(), lost)
    assert torch.equal(out[~lost], clean[~lost])


def silu64(g):
    return g * torch.sigmoid(g)


@pytest.mark.parametrize("T,I,K", [(1, 14336, 4096), (1, 16, 16), (3, 144, 272), (19, 720, 272), (32, 5632, 2048), (33, 128, 4096), (64, 1040, 512), (100, 720, 400), (128, 1792, 1024),
                                   (256, 256, 640), (257, 720, 272), (600, 5632, 2048), (1025, 144, 128), (1025, 3600, 1040), (300, 16, 16)])
def test_gate_up_product(T, I, K):
    g = gen(T + 3 * I + K)
    xq, xs, xv = rows_in_8_bits(rows(g, T, K).double())
    gq, gs, gv = weight(g, I, K)
    uq, us, uv = weight(g, I, K)
    w8 = guarded(torch.cat([gq.view(torch.uint8), uq.view(torch.uint8)]))
    h8, hs = G.empty((T, I), torch.uint8), G.empty((blocks(I), T))
    check(lib().dis_k_gemm_silu_f8(ptr(guarded(xq.view(torch.uint8))), ptr(guarded(xs)), ptr(w8), ptr(guarded(torch.cat([gs, us]))), ptr(h8), ptr(hs), T, I, K, None))
    sync()
    a, b = xv @ gv.T, xv @ uv.T
    oa, ob = sums_off(xv, gv), sums_off(xv, uv)
    want = silu64(a) * b
    # silu' lies in [-0.1, 1.1]; the exponential and the division of the activation are good to a few parts in 10^6 (2^-17)
    near_8_bits(h8, hs, want, 1.1 * oa * (b.abs() + ob) + silu64(a).abs() * ob + want.abs() * 2.0 ** -17)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,H,I", [(1, 4096, 14336), (19, 272, 720), (32, 2048, 5632), (200, 512, 1040), (700, 272, 720)])
def test_feed_forward_block(T, H, I, bf16):
    """One call is its three parts, bit for bit, and each part what it is by itself."""
    g = gen(T + H + I)
    x = rows(g, T, H)
    gq, gs, _ = weight(g, I, H)
    uq, us, _ = weight(g, I, H)
    dq, ds, dv = weight(g, H, I)
    wgu, wgus, wd, wds = guarded(torch.cat([gq, uq]).view(torch.uint8)), guarded(torch.cat([gs, us])), guarded(dq.view(torch.uint8)), guarded(ds)
    x8, xs, h8, hs = G.empty((T, H), torch.uint8), G.empty((blocks(H), T)), G.empty((T, I), torch.uint8), G.empty((blocks(I), T))
    out = G.empty((T, H), torch.bfloat16 if bf16 else torch.float32)
    check(lib().dis_k_ffn_f8(ptr(guarded(x)), ptr(wgu), ptr(wgus), ptr(wd), ptr(wds), ptr(x8), ptr(xs), ptr(h8), ptr(hs), ptr(out), B.BF16 if bf16 else B.F32, T, H, I, None))
    sync()
    q, s = quant(guarded(x))
    assert torch.equal(q, x8) and torch.equal(s, xs)
    h, hsc = G.empty((T, I), torch.uint8), G.empty((blocks(I), T))
    check(lib().dis_k_gemm_silu_f8(ptr(x8), ptr(xs), ptr(wgu), ptr(wgus), ptr(h), ptr(hsc), T, I, H, None))
    sync()
    assert torch.equal(h, h8) and torch.equal(hsc, hs)
    hv = h8.view(F8).double() * hs.double().T.repeat_interleave(128, 1)[:, :I]
    want, bound = hv @ dv.T, sums_off(hv, dv)
    if bf16:
        bound = bound + (want.abs() + bound) * 2.0 ** -8
    assert bool(((out.double() - want).abs() <= bound).all())


def test_empty_calls_and_refusals():
    L, n = lib(), B.ERR_INVALID_ARGUMENT
    a = G.zeros(4096, torch.uint8)
    p, q = ptr(a), ptr(a[1:])
    assert L.dis_k_quant_f8(None, None, None, 0, 128, None) == B.OK
    assert L.dis_k_quant_weight_f8(None, None, None, 0, 128, None) == B.OK
    assert L.dis_k_add_rmsnorm_f8(*[None] * 4, 0, 0, *[None] * 4, 0, 128, 1e-5, None) == B.OK
    for T, N in ((0, 5), (5, 0)):
        assert L.dis_k_gemm_f8(*[None] * 5, B.F32, T, N, 128, None) == B.OK
        assert L.dis_k_gemm_silu_f8(*[None] * 6, T, N * 16, 128, None) == B.OK
    assert L.dis_k_ffn_f8(*[None] * 10, B.F32, 0, 128, 128, None) == B.OK
    for T, K in ((-1, 128), (1, 0), (1, 8), (1, 120), (1, -16), (1 << 30, 16)):
        assert L.dis_k_quant_f8(p, p, p, T, K, None) == n
        assert L.dis_k_add_rmsnorm_f8(p, None, None, None, 0, 0, p, p, p, None, T, K, 1e-5, None) == n
        assert L.dis_k_gemm_f8(p, p, p, p, p, B.F32, T, 16, K, None) == n
        assert L.dis_k_gemm_silu_f8(p, p, p, p, p, p, T, 16, K, None) == n
        assert L.dis_k_ffn_f8(*[p] * 10, B.F32, T, K, 16, None) == n
    for N, K in ((-1, 128), (1 << 30, 16), (5, 24)):
        assert L.dis_k_quant_weight_f8(p, p, p, N, K, None) == n
        assert L.dis_k_gemm_f8(p, p, p, p, p, B.F32, 1, N, K, None) == n
    assert L.dis_k_gemm_silu_f8(p, p, p, p, p, p, 1, 24, 16, None) == n  # inner size
    assert L.dis_k_ffn_f8(*[p] * 10, B.F32, 1, 16, 24, None) == n
    assert L.dis_k_ffn_f8(*[p] * 10, B.F32, 1, 16, 0, None) == n
    assert L.dis_k_add_rmsnorm_f8(p, None, None, None, 0, 0, p, p, p, None, 1, 51216, 1e-5, None) == n
    assert L.dis_k_add_rmsnorm_f8(p, None, None, None, 1, 0, p, p, p, None, 1, 16, 1e-5, None) == n   # partial sums without memory
    assert L.dis_k_add_rmsnorm_f8(p, None, None, p, -1, 0, p, p, p, None, 1, 16, 1e-5, None) == n
    assert L.dis_k_add_rmsnorm_f8(p, p, None, None, 0, 0, p, p, p, None, 1, 16, 1e-5, None) == n      # ids without a table
    assert L.dis_k_add_rmsnorm_f8(p, None, None, p, 2, 18, p, p, p, None, 1, 16, 1e-5, None) == n     # slices off 16 bytes
    assert L.dis_k_gemm_f8(p, p, p, p, p, 7, 1, 16, 16, None) == n
    assert L.dis_k_ffn_f8(*[p] * 10, 7, 1, 16, 16, None) == n
    for k in range(5):
        args = [p] * 5
        args[k] = None
        assert L.dis_k_gemm_f8(*args, B.F32, 1, 16, 16, None) == n
        args[k] = q
        assert L.dis_k_gemm_f8(*args, B.F32, 1, 16, 16, None) == n
    for k in range(6):
        args = [p] * 6
        args[k] = None
        assert L.dis_k_gemm_silu_f8(*args, 1, 16, 16, None) == n
        args[k] = q
        assert L.dis_k_gemm_silu_f8(*args, 1, 16, 16, None) == n
    for k in range(10):
        args = [p] * 10
        args[k] = None
        assert L.dis_k_ffn_f8(*args, B.F32, 1, 16, 16, None) == n
        args[k] = q
        assert L.dis_k_ffn_f8(*args, B.F32, 1, 16, 16, None) == n
    for k in range(3):
        args = [p] * 3
        args[k] = None
        assert L.dis_k_quant_f8(*args, 1, 16, None) == n and L.dis_k_quant_weight_f8(*args, 1, 16, None) == n
        args[k] = q
        assert L.dis_k_quant_f8(*args, 1, 16, None) == n and L.dis_k_quant_weight_f8(*args, 1, 16, None) == n
    sync()
    assert not a.any()


def test_a_captured_feed_forward_replays_with_new_inputs():
    """Captured once on a stream of its own, replayed with other rows in the same memory, beside the same call outside of the graph."""
    T, H, I = 33, 512, 1040
    g = gen(1)
    gq, gs, _ = weight(g, I, H)
    uq, us, _ = weight(g, I, H)
    dq, ds, _ = weight(g, H, I)
    wgu, wgus, wd, wds = guarded(torch.cat([gq, uq]).view(torch.uint8)), guarded(torch.cat([gs, us])), guarded(dq.view(torch.uint8)), guarded(ds)
    x = guarded(rows(g, T, H))
    x8, xs, h8, hs, out = G.empty((T, H), torch.uint8), G.empty((blocks(H), T)), G.empty((T, I), torch.uint8), G.empty((blocks(I), T)), G.empty((T, H))

    def call(o, stream):
        check(lib().dis_k_ffn_f8(ptr(x), ptr(wgu), ptr(wgus), ptr(wd), ptr(wds), ptr(x8), ptr(xs), ptr(h8), ptr(hs), ptr(o), B.F32, T, H, I, stream.cuda_stream))

    st = torch.cuda.Stream()
    call(out, st)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        call(out, torch.cuda.current_stream())
    for i in range(3):
        x.copy_(rows(gen(10 + i), T, H))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        again = G.empty((T, H))
        call(again, torch.cuda.current_stream())
        sync()
        assert torch.equal(out, again)
