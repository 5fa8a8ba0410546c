"""Products in 8-bit floating point where calls meet: chains without a wait between them, several streams, outputs off every boundary, rows of few and odd
blocks, offsets that pass 32 bits."""
import pytest
import torch

from distributed_inference_server_b200 import binding as B
from tests import _gpu_util as G
from tests._gpu_util import DEV, check, lib, ptr, sync
from tests.test_f8_ops_gpu import F8, blocks, gen, guarded, product, rows, rows_in_8_bits, sums_off, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,N,K", [(300, 640, 384), (2100, 5008, 384), (2100, 5008, 128), (129, 144, 128), (255, 256, 640), (511, 272, 16), (1300, 8192, 1152), (2048, 8192, 144),
                                   (257, 20000, 256), (16, 128, 384), (128, 1000, 896), (300, 1001, 384), (700, 33, 640), (2100, 5003, 272), (257, 129, 16), (1025, 4143, 384)])
@pytest.mark.parametrize("bf16,by", [(False, 1), (True, 1), (True, 8), (False, 4)])
def test_outputs_that_start_anywhere(T, N, K, bf16, by):
    """Outputs that start `by` elements behind a boundary, rows of odd and even lengths: narrower vectors, words that two features share, single elements; odd and even numbers of
    blocks."""
    g = gen(T + N + K)
    xq, xs, xv = rows_in_8_bits(rows(g, T, K).double())
    wq, ws, wv = weight(g, N, K)
    flat = G.empty((T * N + 64,), torch.bfloat16 if bf16 else torch.float32)
    flat.fill_(7.0)
    out = flat[by:by + T * N].view(T, N)
    check(lib().dis_k_gemm_f8(ptr(guarded(xq.view(torch.uint8))), ptr(guarded(xs)), ptr(guarded(wq.view(torch.uint8))), ptr(guarded(ws)), ptr(out), B.BF16 if bf16 else B.F32, T, N, K,
                              None))
    sync()
    want, bound = xv @ wv.T, sums_off(xv, wv)
    if bf16:
        bound = bound + (want.abs() + bound) * 2.0 ** -8
    assert bool(((out.double() - want).abs() <= bound).all())
    assert bool((flat[:by] == 7).all()) and bool((flat[by + T * N:] == 7).all())


@pytest.mark.parametrize("T,N,K", [(1, 512, 512), (40, 640, 1040), (200, 512, 1024), (700, 1280, 512)])
def test_chains_without_a_wait(T, N, K):
    """Weights and rows turned into 8 bits and multiplied right behind, over and over in the same memory with other numbers: what a product reads is what the calls in
    front of it wrote."""
    g = gen(N + K)
    w = [(torch.randn(N, K, generator=g, device=DEV) * 0.05).to(torch.bfloat16) for _ in range(3)]
    x = [rows(g, T, K) for _ in range(3)]
    xb, wb = guarded(x[0]), guarded(w[0])
    x8, xs, w8, ws = G.empty((T, K), torch.uint8), G.empty((blocks(K), T)), G.empty((N, K), torch.uint8), G.empty((blocks(N), blocks(K)))
    outs = [G.empty((T, N)) for _ in range(30)]
    L = lib()

    def call(i, wait):
        xb.copy_(x[i % 3])
        wb.copy_(w[(i // 2) % 3])
        for f, a in ((L.dis_k_quant_weight_f8, (ptr(wb), ptr(w8), ptr(ws), N, K, None)), (L.dis_k_quant_f8, (ptr(xb), ptr(x8), ptr(xs), T, K, None)),
                     (L.dis_k_gemm_f8, (ptr(x8), ptr(xs), ptr(w8), ptr(ws), ptr(outs[i]), B.F32, T, N, K, None))):
            check(f(*a))
            if wait:
                sync()

    for i in range(30):
        call(i, False)
    sync()
    got = [o.clone() for o in outs]
    for i in range(6):
        call(i, True)
    for i in range(30):
        assert torch.equal(got[i], outs[i % 6]), i  # (the numbers repeat every six calls)


def test_a_layer_in_a_chain():
    """Norm, projection, norm of the sum, feed-forward block: as a decoder layer strings them together, against the same with a wait behind every call."""
    T, H, I = 48, 512, 1040
    g = gen(3)
    wq = guarded((torch.randn(H, H, generator=g, device=DEV) * 0.05).to(torch.bfloat16))
    wgu = guarded((torch.randn(2 * I, H, generator=g, device=DEV) * 0.05).to(torch.bfloat16))
    wd = guarded((torch.randn(H, I, generator=g, device=DEV) * 0.05).to(torch.bfloat16))
    gain = guarded(torch.rand(H, generator=g, device=DEV) + 0.5)
    L = lib()
    q8, qs = G.empty((H, H), torch.uint8), G.empty((4, 4))
    gu8, gus = G.empty((2 * I, H), torch.uint8), G.empty((2 * blocks(I), 4))
    d8, ds = G.empty((H, I), torch.uint8), G.empty((4, blocks(I)))
    check(L.dis_k_quant_weight_f8(ptr(wq), ptr(q8), ptr(qs), H, H, None))
    for part in range(2):  # the gate's blocks, then the up's
        check(L.dis_k_quant_weight_f8(ptr(wgu[part * I:]), ptr(gu8[part * I:]), ptr(gus[part * blocks(I):]), I, H, None))
    check(L.dis_k_quant_weight_f8(ptr(wd), ptr(d8), ptr(ds), H, I, None))
    x0 = torch.randn(T, H, generator=g, device=DEV)
    results = []
    for wait in (True, False, False, False):
        x = guarded(x0)
        x8, xs, h8, hs, part = G.empty((T, H), torch.uint8), G.empty((4, T)), G.empty((T, I), torch.uint8), G.empty((blocks(I), T)), G.empty((T, H))
        calls = [lambda: L.dis_k_add_rmsnorm_f8(ptr(x), None, None, None, 0, 0, ptr(gain), ptr(x8), ptr(xs), None, T, H, 1e-5, None)]
        for _ in range(5):
            calls += [lambda: L.dis_k_gemm_f8(ptr(x8), ptr(xs), ptr(q8), ptr(qs), ptr(part), B.F32, T, H, H, None),
                      lambda: L.dis_k_add_rmsnorm_f8(ptr(x), None, None, ptr(part), 1, 0, ptr(gain), ptr(x8), ptr(xs), None, T, H, 1e-5, None),
                      lambda: L.dis_k_gemm_silu_f8(ptr(x8), ptr(xs), ptr(gu8), ptr(gus), ptr(h8), ptr(hs), T, I, H, None),
                      lambda: L.dis_k_gemm_f8(ptr(h8), ptr(hs), ptr(d8), ptr(ds), ptr(part), B.F32, T, H, I, None),
                      lambda: L.dis_k_add_rmsnorm_f8(ptr(x), None, None, ptr(part), 1, 0, ptr(gain), ptr(x8), ptr(xs), None, T, H, 1e-5, None)]
        for c in calls:
            check(c())
            if wait:
                sync()
        sync()
        results.append(x.clone())
    assert bool(results[0].isfinite().all()) and not torch.equal(results[0], x0)
    assert all(torch.equal(r, results[0]) for r in results[1:])


def test_calls_on_several_streams():
    """Products of different sizes on three streams at once are what they are alone."""
    sizes = [(32, 2048, 2048), (300, 1024, 1040), (1, 4096, 4096), (700, 512, 2048), (64, 1000, 272)]
    g = gen(9)
    state = []
    for T, N, K in sizes:
        xq, xs, _ = rows_in_8_bits(rows(g, T, K).double())
        wq, ws, _ = weight(g, N, K)
        state.append((guarded(xq.view(torch.uint8)), guarded(xs), guarded(wq.view(torch.uint8)), guarded(ws), T, N, K))
    alone = []
    for a in state:
        alone.append(product(*a))
        sync()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [[G.empty((a[4], a[5])) for a in state] for _ in streams]
    sync()
    for k, st in enumerate(streams):
        for i in range(len(state)):
            a = state[(i + k) % len(state)]
            check(lib().dis_k_gemm_f8(ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(a[3]), ptr(outs[k][(i + k) % len(state)]), B.F32, a[4], a[5], a[6], st.cuda_stream))
    sync()
    for o in outs:
        assert all(torch.equal(x, y) for x, y in zip(o, alone))


def test_offsets_past_32_bits():
    """Outputs, weights and rows of more than 2^31 entries: the last rows are what they are by themselves."""
    g = gen(1)
    T, N, K = 40000, 60000, 16  # an output of 2.4e9 entries
    xq, xs, xv = rows_in_8_bits(rows(g, T, K).double())
    wq, ws, wv = weight(g, N, K)
    out = torch.empty(T, N, dtype=torch.bfloat16, device=DEV)
    check(lib().dis_k_gemm_f8(ptr(xq.view(torch.uint8)), ptr(xs), ptr(wq.view(torch.uint8)), ptr(ws), ptr(out), B.BF16, T, N, K, None))
    sync()
    for r in (slice(0, 3), slice(T - 3, T), slice(T * 9 // 10, T * 9 // 10 + 2)):
        want, bound = xv[r] @ wv.T, sums_off(xv[r], wv)
        bound = bound + (want.abs() + bound) * 2.0 ** -8
        assert bool(((out[r].double() - want).abs() <= bound).all())
    del out, wv
    T, N, K = 3, 140000, 16384  # a weight of 2.3e9
    w8 = torch.randint(0, 0x7e, (N, K), dtype=torch.uint8, device=DEV)
    ws = torch.rand(blocks(N), blocks(K), device=DEV)
    xq, xs, xv = rows_in_8_bits(rows(g, T, K).double())
    out = torch.empty(T, N, device=DEV)
    check(lib().dis_k_gemm_f8(ptr(xq.view(torch.uint8)), ptr(xs), ptr(w8), ptr(ws), ptr(out), B.F32, T, N, K, None))
    sync()
    for r in (slice(0, 2), slice(N - 130, N)):
        wv = w8[r].view(F8).double() * ws.repeat_interleave(128, 0)[:N][r].repeat_interleave(128, 1).double()
        assert bool(((out[:, r].double() - xv @ wv.T).abs() <= sums_off(xv, wv)).all())
    del w8, out
    T, K = 140000, 16384  # rows of 2.3e9
    x = torch.empty(T, K, dtype=torch.bfloat16, device=DEV)
    x[-5:] = rows(g, 5, K)
    x[:5] = x[-5:]
    x8, s = torch.empty(T, K, dtype=torch.uint8, device=DEV), torch.empty(blocks(K), T, device=DEV)
    check(lib().dis_k_quant_f8(ptr(x), ptr(x8), ptr(s), T, K, None))
    sync()
    q, want, _ = rows_in_8_bits(x[-5:].double())
    assert torch.equal(x8[-5:], q.view(torch.uint8)) and torch.equal(s[:, -5:], want) and torch.equal(x8[:5], x8[-5:])
    del x, x8, s
    T, H = 530000, 4096   # a residual of 2.2e9
    x, ids = torch.empty(T, H, device=DEV), torch.zeros(T, dtype=torch.int32, device=DEV)
    ids[-3:] = torch.tensor([1, 2, 3], device=DEV)
    embed, gain = torch.randn(4, H, generator=g, device=DEV).to(torch.bfloat16), torch.ones(H, device=DEV)
    x8, s = torch.empty(T, H, dtype=torch.uint8, device=DEV), torch.empty(blocks(H), T, device=DEV)
    check(lib().dis_k_add_rmsnorm_f8(ptr(x), ptr(ids), ptr(embed), None, 0, 0, ptr(gain), ptr(x8), ptr(s), None, T, H, 1e-5, None))
    sync()
    small, s8, ss = G.empty((4, H)), G.empty((4, H), torch.uint8), G.empty((blocks(H), 4))
    check(lib().dis_k_add_rmsnorm_f8(ptr(small), ptr(torch.arange(4, dtype=torch.int32, device=DEV)), ptr(embed), None, 0, 0, ptr(gain), ptr(s8), ptr(ss), None, 4, H, 1e-5, None))
    sync()
    assert torch.equal(x[-3:], embed[1:].float())
    v = lambda q, sc: q.view(F8).float() * sc.T.repeat_interleave(128, 1)  # noqa: E731
    a, b = v(x8[-3:], s[:, -3:]), v(s8[1:], ss[:, 1:])
    # (256 threads a row there, 1024 here: the mean is summed in another order, and a value on the border of two e4m3 numbers may fall either way)
    assert bool(((a - b).abs() <= b.abs() * 2.0 ** -3 + ss[:, 1:].T.repeat_interleave(128, 1) * 2.0 ** -9).all()) and float((a != b).float().mean()) < 1e-3
