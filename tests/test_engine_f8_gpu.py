"""Engines whose layers' projections are in 8-bit floating point (DIS_FLAG_WEIGHTS_F8), end to end through the C ABI, against a restatement of the decoder
whose weights and projection inputs pass through the same 8 bits.

The tolerance: values that the two sides know differently by however little may be rounded to neighbouring e4m3 numbers.  If every rounding of a projection's
input fell independently, each would be off by a step (on average 2^-3.5 of the value) over the root of 12, on both sides: 0.036 of the sublayer's result,
rms.  A sublayer passes the noise of what it reads on and adds its own: 0.036 sqrt(2 L) after L layers.  The largest of a thousand logits' noise is
four times its rms, the largest logit 3.5 times theirs: 0.036 sqrt(2 L) 4 / 3.5 of max|logit|, 0.101 for three layers and 0.082 for two.  (The restatement against itself
with its projections' inputs moved by one part in 2^22: up to 0.058 and 0.049.)
"""
import numpy as np
import pytest
import torch

from distributed_inference_server_b200 import Engine, InferenceParams, WorkerConfig, WorkerError
from distributed_inference_server_b200 import binding as B
from oracle import oracle as O
from tests._gpu_util import to_engine_shape
from tests.test_engine_cache_gpu import Restated, bf16, follow
from tests.test_engine_gpu import make_engine, rel_err

pytestmark = pytest.mark.gpu
def tol(shape):
    return 0.036 * (2 * shape.layers) ** 0.5 * 4 / 3.5


SMALL = O.ModelShape(1024, 256, 3, 8, 2, 64, 704, 512)
WIDE = O.ModelShape(1024, 272, 2, 8, 2, 128, 1040, 512)   # widths that end inside a block of 128


def rounded(x, dims):
    """fp32 values in e4m3 under a power of two for each block of 128 of the last dimension (dims = 1) or of the last two."""
    n, k = x.shape
    pad = torch.nn.functional.pad(x, (0, -k % 128, 0, -n % 128 if dims == 2 else 0))
    b = pad.view(-1, 128 if dims == 2 else 1, pad.shape[1] // 128, 128)
    top = b.abs().amax((1, 3), keepdim=True)
    m, e = torch.frexp(top / 448)
    s = torch.ldexp(torch.ones_like(m), e - (m == 0.5).int()).clamp_min(2.0 ** -126)
    return ((b / s).to(torch.float8_e4m3fn).float() * s).view(pad.shape)[:n, :k].contiguous()


class RestatedF8(Restated):
    def __init__(self, shape, seed):
        super().__init__(shape, seed)
        for (k, l), a in list(self.t.items()):
            if k in (O.WQ, O.WK, O.WV, O.WO, O.WGATE, O.WUP, O.WDOWN):
                self.t[k, l] = rounded(a, 2)

    def logits(self, tokens):
        s, d = self.s, self.s.head_dim
        n, group = len(tokens), s.n_heads // s.n_kv_heads
        plain = lambda x, g: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s.rms_eps) * g  # noqa: E731
        x = self.t[O.EMBED, 0][torch.tensor(tokens)]
        a = torch.arange(n, dtype=torch.float64)[:, None] * s.rope_theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        c, sn = a.cos().float()[:, None], a.sin().float()[:, None]
        for l in range(s.layers):
            w = lambda k: self.t[k, l]  # noqa: E731
            h = rounded(plain(x, w(O.ATTN_NORM)), 1)
            q, k, v = ((h @ w(i).T).view(n, -1, d) for i in (O.WQ, O.WK, O.WV))
            turn = lambda y: torch.cat([y[..., :d // 2] * c - y[..., d // 2:] * sn, y[..., d // 2:] * c + y[..., :d // 2] * sn], -1)  # noqa: E731
            q, k, v = bf16(turn(q)), bf16(turn(k)), bf16(v)
            k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
            p = torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5
            p = torch.softmax(p.masked_fill(torch.ones(n, n).triu(1).bool(), -torch.inf), -1)
            x = x + rounded(bf16(torch.einsum("hqk,khd->qhd", p, v).reshape(n, -1)), 1) @ w(O.WO).T
            h = rounded(plain(x, w(O.MLP_NORM)), 1)
            x = x + rounded(torch.nn.functional.silu(h @ w(O.WGATE).T) * (h @ w(O.WUP).T), 1) @ w(O.WDOWN).T
        return (self.norm(x, self.t[O.FINAL_NORM, 0]) @ self.t[O.LM_HEAD, 0].T).numpy()


def bits(x):
    return (x.to(torch.bfloat16).view(torch.int16).numpy().astype(np.int32) & 0xffff).astype(np.uint16)


@pytest.mark.parametrize("shape", [SMALL, WIDE], ids=["d64", "d128"])
@pytest.mark.parametrize("flags", [0, B.FLAG_NO_GRAPH | B.FLAG_NO_PDL], ids=["graph", "eager"])
def test_f8_engine_follows_its_restatement(shape, flags):
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, shape.vocab, n).tolist() for n in (5, 33, 300, 16)]
    e = make_engine(shape, seed=7, page_size=16, flags=flags | B.FLAG_WEIGHTS_F8)  # (chunks of 256 tokens: products in tiles and in pairs)
    _, out, logits = follow(e, prompts, 6)
    ref = RestatedF8(shape, 7)
    for i, p in enumerate(prompts):
        want = ref.logits(p + out[i])
        for k in range(6):
            assert rel_err(logits[k][i], want[len(p) + k]) <= tol(shape), (i, k)
        row = want[len(p) - 1]  # the prompt's own last row: its greedy choice, but for near ties
        assert row.max() - row[out[i][0]] <= tol(shape) * np.abs(row).max(), i
    e.close()


@pytest.mark.parametrize("how", ["synthetic", "loaded", "loaded_bf16"])
def test_weights_are_what_their_8_bits_stand_for(how):
    """Loaded or generated, every tensor reads back as the values that 8 bits hold, exactly in bf16; what is not a projection is as it was."""
    m = O.Oracle(WIDE, act_round=True)
    m.fill_synthetic(3, True)
    if how == "synthetic":
        e = make_engine(WIDE, seed=3, flags=B.FLAG_WEIGHTS_F8)
    else:
        e = Engine(WorkerConfig(to_engine_shape(WIDE), max_batch=8, kv_pages=64, page_size=16, max_step_tokens=256, flags=B.FLAG_WEIGHTS_F8))
        for kind, layer, a in m.tensors():
            a = np.array(a, np.float32)
            e.load_tensor(kind, layer, bits(torch.from_numpy(a)) if how == "loaded_bf16" else a)
        e.finalize()
    for kind, layer, a in m.tensors():
        a = torch.from_numpy(np.array(a, np.float32)).view(1, -1) if np.ndim(a) == 1 else torch.from_numpy(np.array(a, np.float32))
        want = rounded(bf16(a), 2) if kind in (O.WQ, O.WK, O.WV, O.WO, O.WGATE, O.WUP, O.WDOWN) else a
        assert np.array_equal(e.read_tensor(kind, layer), bits(want).reshape(-1)), (kind, layer)
    e.close()


def test_weights_that_are_in_8_bits_already():
    """Tensors of a checkpoint in 8 bits with scales of its own (max / 448, no powers of two) give the logits of what they stand for, and read back as that."""
    ref = RestatedF8(WIDE, 5)
    m = O.Oracle(WIDE, act_round=True)
    m.fill_synthetic(5, True)
    e = Engine(WorkerConfig(to_engine_shape(WIDE), max_batch=8, kv_pages=64, page_size=16, max_step_tokens=256, flags=B.FLAG_WEIGHTS_F8))
    for kind, layer, a in m.tensors():
        a = torch.from_numpy(np.array(a, np.float32))
        if kind not in (O.WQ, O.WK, O.WV, O.WO, O.WGATE, O.WUP, O.WDOWN):
            e.load_tensor(kind, layer, a.numpy())
            continue
        n, k = a.shape
        pad = torch.nn.functional.pad(a, (0, -k % 128, 0, -n % 128))
        b = pad.view(-1, 128, pad.shape[1] // 128, 128)
        s = b.abs().amax((1, 3)) / 448
        q = (b / s[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        value = (q.float() * s[:, None, :, None]).view(pad.shape)[:n, :k].contiguous()
        e.load_tensor_f8(kind, layer, q.view(pad.shape)[:n, :k].contiguous().view(torch.uint8).numpy(), s.numpy())
        assert np.array_equal(e.read_tensor(kind, layer), bits(value).reshape(-1)), (kind, layer)
        ref.t[kind, layer] = value
    e.finalize()
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, WIDE.vocab, n).tolist() for n in (12, 200)]
    _, out, logits = follow(e, prompts, 3)
    for i, p in enumerate(prompts):
        want = ref.logits(p + out[i])
        for k in range(3):
            assert rel_err(logits[k][i], want[len(p) + k]) <= tol(WIDE), (i, k)
    q = np.zeros((WIDE.hidden, WIDE.inter), np.uint8)
    s = np.zeros((-(-WIDE.hidden // 128), -(-WIDE.inter // 128)), np.float32)
    for kind, layer in ((O.EMBED, 0), (O.LM_HEAD, 0), (O.ATTN_NORM, 0), (O.WDOWN, 2), (O.WDOWN, -1), (77, 0)):
        with pytest.raises(WorkerError):
            e.load_tensor_f8(kind, layer, q, s)
    with pytest.raises(TypeError):
        e.load_tensor_f8(O.WDOWN, 0, q, s[:, 1:])
    e.close()
    e = make_engine(WIDE, seed=1)
    with pytest.raises(WorkerError) as err:
        e.load_tensor_f8(O.WDOWN, 0, q, s)
    assert "DIS_FLAG_WEIGHTS_F8" in str(err.value)
    e.close()


def test_f8_engine_mixed_passes():
    """Prompts read in chunks beside running sequences: the restatement's choices."""
    rng = np.random.default_rng(2)
    a, b = (rng.integers(0, SMALL.vocab, n).tolist() for n in (40, 90))
    e = make_engine(SMALL, seed=9, page_size=16, flags=B.FLAG_WEIGHTS_F8)
    P = InferenceParams(max_tokens=30, temperature=0.0)
    s = e.seq_add(a, P)
    toks, _ = e.prefill([s])
    got = [int(toks[0])]
    t = e.seq_add(b, P)
    first = None
    for _ in range(6):
        toks, fin, made = e.step([s, t], 25)
        got.append(int(toks[0]))
        if made[1] and first is None:
            first = e.last_logits(2)[1].copy()
    ref = RestatedF8(SMALL, 9)
    assert first is not None and rel_err(first, ref.logits(b)[-1]) <= tol(SMALL)
    want = ref.logits(a + got)
    for k, g in enumerate(got):  # the greedy choice, but for near ties
        row = want[len(a) - 1 + k]
        assert row.max() - row[g] <= tol(SMALL) * np.abs(row).max(), k
    e.close()


def test_every_way_through_a_step_gives_the_same_logits():
    """Decode steps from a graph and launched one by one are the same kernels on the same numbers: equal bits.  Beside the 8-bit cache and shared
    prefixes the engine follows the engine without them."""
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, SMALL.vocab, n).tolist() for n in (9, 60, 31)]
    runs = {}
    for name, flags in (("graph", 0), ("eager", B.FLAG_NO_GRAPH), ("plain", B.FLAG_NO_GRAPH | B.FLAG_NO_PDL), ("cache", B.FLAG_KV_INT8 | B.FLAG_ATTN_SHARED | B.FLAG_PREFIX_CACHE)):
        e = make_engine(SMALL, seed=11, page_size=16, flags=flags | B.FLAG_WEIGHTS_F8)
        _, out, logits = follow(e, prompts, 4)
        runs[name] = (out, logits)
        e.close()
    for name in ("eager", "plain"):
        assert runs[name][0] == runs["graph"][0]
        assert all(np.array_equal(x, y) for x, y in zip(runs[name][1], runs["graph"][1])), name
    for i in range(3):
        for k in range(4):
            if runs["cache"][0][i][:k + 1] != runs["graph"][0][i][:k + 1]:
                break  # another token at a near tie
            assert rel_err(runs["cache"][1][k][i], runs["graph"][1][k][i]) <= tol(SMALL), (i, k)


def test_weights_take_half_the_memory():
    shape = O.ModelShape(1024, 2048, 8, 16, 4, 128, 5632, 1 << 16)
    used = []
    for flags in (0, B.FLAG_WEIGHTS_F8):
        e = Engine(WorkerConfig(to_engine_shape(shape), max_batch=4, kv_pages=16, page_size=64, max_step_tokens=128, flags=flags))
        used.append(e.status().memory_used)
        e.close()
    weights = 8 * (2 * 2048 * 2048 + 2 * 512 * 2048 + 3 * 2048 * 5632)
    assert 0.9 * weights < used[0] - used[1] < weights, (used, weights)  # two bytes an entry and one, less a tensor on its way and the rows in 8 bits


def test_refused_where_it_cannot_be():
    def attempt(shape, **kw):
        with pytest.raises(WorkerError) as err:
            Engine(WorkerConfig(to_engine_shape(shape), max_batch=2, kv_pages=8, page_size=16, **kw))
        return str(err.value)
    assert "multiples of" in attempt(O.ModelShape(1024, 256, 1, 6, 1, 64, 704, 256), flags=B.FLAG_WEIGHTS_F8)
    assert "multiples of" in attempt(O.ModelShape(1024, 264, 1, 8, 2, 64, 704, 256), flags=B.FLAG_WEIGHTS_F8)
    assert "multiples of" in attempt(O.ModelShape(1024, 256, 1, 8, 2, 64, 712, 256), flags=B.FLAG_WEIGHTS_F8)
    assert "GEMV" in attempt(SMALL, flags=B.FLAG_WEIGHTS_F8 | B.FLAG_FORCE_GEMV)
    from distributed_inference_server_b200 import models
    spec = models.nifulix_spec({"architecture": "Nifulix", "vocab": 256, "width": 128, "norm": {"eps": 1e-5}, "residual_mult": 0.5, "layers": [
        {"type": "retention", "mixer": {"heads": 1, "dim": 128, "vdim": 128, "rot": {"base": 10000.0, "dims": 128}, "decay": [0.9]}, "mlp": {"kind": "dense", "ff": 256}}]})
    with pytest.raises(WorkerError) as err:
        Engine(WorkerConfig(None, stack=spec, max_batch=2, context_size=256, flags=B.FLAG_WEIGHTS_F8))
    assert "Llama family" in str(err.value)
