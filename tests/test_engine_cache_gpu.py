"""Engines that keep keys and values in 8 bits (DIS_FLAG_KV_INT8) and engines whose decode steps read common pages once (DIS_FLAG_ATTN_SHARED), end to
end through the C ABI: against a restatement of the decoder whose keys and values pass through 8 bits, and against engines without the flags.  The
tolerance is the one of the other engine tests: 2e-2 of max|logit|."""
import numpy as np
import pytest
import torch

from distributed_inference_server_b200 import Engine, InferenceParams, WorkerConfig, WorkerError
from distributed_inference_server_b200 import binding as B
from oracle import oracle as O
from tests._gpu_util import to_engine_shape
from tests.test_engine_gpu import make_engine, rel_err

pytestmark = pytest.mark.gpu
TOL = 2e-2
SMALL = O.ModelShape(1024, 256, 3, 8, 2, 64, 704, 512)
WIDE = O.ModelShape(1024, 256, 2, 8, 2, 128, 704, 512)


def bf16(x):
    return x.to(torch.bfloat16).float()


class Restated:
    """The decoder in fp32 with the engine's bf16 rounding points, keys and values as 8-bit rows."""

    def __init__(self, shape, seed):
        self.s = shape
        m = O.Oracle(shape, act_round=True)
        m.fill_synthetic(seed, True)
        self.t = {(k, l if k in O.PER_LAYER else 0): torch.from_numpy(np.array(a, np.float32)) for k, l, a in m.tensors()}

    def norm(self, x, g):
        return bf16(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.s.rms_eps) * g)

    def logits(self, tokens):
        s, d = self.s, self.s.head_dim
        n, group = len(tokens), s.n_heads // s.n_kv_heads
        x = self.t[O.EMBED, 0][torch.tensor(tokens)]
        a = torch.arange(n, dtype=torch.float64)[:, None] * s.rope_theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        c, sn = a.cos().float()[:, None], a.sin().float()[:, None]
        for l in range(s.layers):
            w = lambda k: self.t[k, l]  # noqa: E731
            h = self.norm(x, w(O.ATTN_NORM))
            q, k, v = ((h @ w(i).T).view(n, -1, d) for i in (O.WQ, O.WK, O.WV))
            turn = lambda y: torch.cat([y[..., :d // 2] * c - y[..., d // 2:] * sn, y[..., d // 2:] * c + y[..., :d // 2] * sn], -1)  # noqa: E731
            q, k = bf16(turn(q)), turn(k)
            k, v = (torch.round(y / (y.abs().amax(-1, keepdim=True) / 127)) * (y.abs().amax(-1, keepdim=True) / 127) for y in (k, v))
            k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
            p = torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5
            p = torch.softmax(p.masked_fill(torch.ones(n, n).triu(1).bool(), -torch.inf), -1)
            o = bf16(torch.einsum("hqk,khd->qhd", p, v).reshape(n, -1))
            x = x + o @ w(O.WO).T
            h = self.norm(x, w(O.MLP_NORM))
            x = x + bf16(torch.nn.functional.silu(h @ w(O.WGATE).T) * (h @ w(O.WUP).T)) @ w(O.WDOWN).T
        return (self.norm(x, self.t[O.FINAL_NORM, 0]) @ self.t[O.LM_HEAD, 0].T).numpy()


def follow(e, prompts, steps):
    """Greedy continuations and the logits of every decode step."""
    P = InferenceParams(max_tokens=steps + 2, temperature=0.0)
    slots = [e.seq_add(p, P) for p in prompts]
    toks, _ = e.prefill(slots)
    out, logits = [[int(t)] for t in toks], []
    for _ in range(steps):
        toks, _ = e.decode(slots)
        logits.append(e.last_logits(len(slots)).copy())
        for o, t in zip(out, toks):
            o.append(int(t))
    return slots, out, logits


@pytest.mark.parametrize("shape", [SMALL, WIDE], ids=["d64", "d128"])
@pytest.mark.parametrize("flags", [0, B.FLAG_NO_GRAPH | B.FLAG_NO_PDL], ids=["graph", "eager"])
def test_int8_engine_follows_its_restatement(shape, flags):
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, shape.vocab, n).tolist() for n in (5, 33, 100, 16)]
    e = make_engine(shape, seed=7, page_size=16, max_step_tokens=64, flags=flags | B.FLAG_KV_INT8)  # (prompts in chunks of 64)
    _, out, logits = follow(e, prompts, 6)
    ref = Restated(shape, 7)
    for i, p in enumerate(prompts):
        want = ref.logits(p + out[i])
        for k in range(6):
            assert rel_err(logits[k][i], want[len(p) + k]) <= TOL, (i, k)
        row = want[len(p) - 1]  # the prompt's own last row: its greedy choice, but for near ties
        assert row.max() - row[out[i][0]] <= TOL * np.abs(row).max(), i
    e.close()


def test_int8_engine_mixed_passes():
    """Prompts read in chunks beside running sequences: the same logits as one after the other."""
    rng = np.random.default_rng(2)
    a, b = (rng.integers(0, SMALL.vocab, n).tolist() for n in (40, 90))
    e = make_engine(SMALL, seed=9, page_size=16, flags=B.FLAG_KV_INT8)
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
    ref = Restated(SMALL, 9)
    assert first is not None and rel_err(first, ref.logits(b)[-1]) <= TOL
    want = ref.logits(a + got)
    for k, g in enumerate(got):  # the greedy choice, but for near ties
        row = want[len(a) - 1 + k]
        assert row.max() - row[g] <= TOL * np.abs(row).max(), k
    e.close()


def test_int8_engine_has_about_twice_the_pages():
    pages = []
    for flags in (0, B.FLAG_KV_INT8):
        e = Engine(WorkerConfig(to_engine_shape(O.ModelShape(1024, 256, 16, 8, 2, 128, 704, 1 << 16)), max_batch=512, page_size=64, max_step_tokens=512, kv_mem_fraction=0.02,
                                flags=flags))
        pages.append(e.status().kv_pages_total)
        e.close()
    assert 1.7 < pages[1] / pages[0] < 2.0, pages


@pytest.mark.parametrize("int8", [False, True])
def test_common_pages_are_read_once(int8):
    """Requests behind one prompt, its pages shared by the prefix cache: with DIS_FLAG_ATTN_SHARED the decode steps launch the shared attention (two kernels
    more per layer, one less where the pages are bf16 and written by the attention) and give the same logits."""
    shape = O.ModelShape(1024, 256, 2, 32, 8, 128, 704, 2048)
    rng = np.random.default_rng(3)
    base = rng.integers(0, shape.vocab, 1300).tolist()
    prompts = [base + rng.integers(0, shape.vocab, 3 + 5 * i).tolist() for i in range(32)]
    assert B.load().dis_k_attn_shared_in_common(32, 32, 8, 128, 1296, int8) == 1
    runs = []
    for shared in (0, B.FLAG_ATTN_SHARED):
        e = make_engine(shape, seed=5, max_batch=32, kv_pages=500, page_size=16, max_step_tokens=4096, flags=B.FLAG_PREFIX_CACHE | shared | (B.FLAG_KV_INT8 if int8 else 0))
        P = InferenceParams(max_tokens=20, temperature=0.0)
        e.seq_remove(follow(e, [base], 0)[0][0])  # the base's pages are in the cache
        slots = [e.seq_add(p, P) for p in prompts]
        toks, _ = e.prefill(slots)
        history, logits, launches = [[int(t)] for t in toks], [], []
        for k in range(4):
            before = e.status().kernel_launches
            toks, _ = e.decode(slots)
            launches.append(e.status().kernel_launches - before)
            logits.append(e.last_logits(32).copy())
            for h, t in zip(history, toks):
                h.append(int(t))
        # without the first requests nothing changes for the others; two are too few to share
        toks, _ = e.decode(slots[:2])
        few = e.status().kernel_launches
        runs.append((history, logits, launches))
        assert few > 0
        e.close()
    extra = {a - b for a, b in zip(runs[1][2], runs[0][2])}
    assert extra == {2 * (2 if int8 else 3)}, extra  # 8 bits: 1 + 1 -> 1 + 3 kernels in each of two layers; bf16: 1 -> 1 + 3
    for i in range(32):
        for k in range(4):
            if runs[0][0][i][:k + 1] != runs[1][0][i][:k + 1]:
                break  # another token at a near tie: the histories differ from here on
            assert rel_err(runs[1][1][k][i], runs[0][1][k][i]) <= TOL, (i, k)
    same = sum(a == b for a, b in zip(runs[0][0], runs[1][0]))
    assert same >= 24, same


def test_refused_where_it_cannot_be():
    with pytest.raises(WorkerError) as err:
        Engine(WorkerConfig(to_engine_shape(O.ModelShape(1024, 256, 1, 6, 2, 64, 704, 256)), max_batch=2, kv_pages=8, page_size=16, flags=B.FLAG_KV_INT8))
    assert "query heads per kv head" in str(err.value)
    from tests import _nifulix_util  # noqa: F401  (a layer-list design)
    from distributed_inference_server_b200 import models
    spec = models.nifulix_spec({"architecture": "Nifulix", "vocab": 256, "width": 128, "norm": {"eps": 1e-5}, "residual_mult": 0.5, "layers": [
        {"type": "retention", "mixer": {"heads": 1, "dim": 128, "vdim": 128, "rot": {"base": 10000.0, "dims": 128}, "decay": [0.9]}, "mlp": {"kind": "dense", "ff": 256}}]})
    for flag in (B.FLAG_KV_INT8, B.FLAG_ATTN_SHARED):
        with pytest.raises(WorkerError) as err:
            Engine(WorkerConfig(None, stack=spec, max_batch=2, context_size=256, flags=flag))
        assert "Llama family" in str(err.value)
