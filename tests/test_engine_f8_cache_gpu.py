"""Engines with 8-bit projections beside shared prefixes and the 8-bit cache: requests behind one prompt against a restatement on the requests' own tokens, and
proof that their decode steps read the common pages once.

The tolerance is the sum of the two that the flags have by themselves: 0.036 sqrt(2 L) 4 / 3.5 of max|logit| (test_engine_f8_gpu.py) and 2e-2 (test_engine_cache_gpu.py)."""
import numpy as np
import pytest
import torch

from distributed_inference_server_b200 import InferenceParams
from distributed_inference_server_b200 import binding as B
from oracle import oracle as O
from tests.test_engine_cache_gpu import TOL, bf16, follow
from tests.test_engine_f8_gpu import RestatedF8, rounded, tol
from tests.test_engine_gpu import make_engine, rel_err

pytestmark = pytest.mark.gpu
SHAPE = O.ModelShape(1024, 256, 2, 32, 8, 128, 704, 2048)
LIMIT = tol(SHAPE) + TOL


class RestatedBoth(RestatedF8):
    """With keys and values as 8-bit rows too where the engine keeps them so."""

    def __init__(self, shape, seed, int8):
        super().__init__(shape, seed)
        self.int8 = int8

    def kept(self, y):
        if not self.int8:
            return bf16(y)
        s = y.abs().amax(-1, keepdim=True) / 127
        return torch.round(y / s) * s

    def logits(self, tokens, rows):
        """Of the last `rows` positions"""
        s, d = self.s, self.s.head_dim
        n, group = len(tokens), s.n_heads // s.n_kv_heads
        plain = lambda x, g: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s.rms_eps) * g  # noqa: E731
        x = self.t[O.EMBED, 0][torch.tensor(tokens)]
        a = torch.arange(n, dtype=torch.float64)[:, None] * s.rope_theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        c, sn = a.cos().float()[:, None], a.sin().float()[:, None]
        turn = lambda y: torch.cat([y[..., :d // 2] * c - y[..., d // 2:] * sn, y[..., d // 2:] * c + y[..., :d // 2] * sn], -1)  # noqa: E731
        later = torch.ones(n, n).triu(1).bool()
        for l in range(s.layers):
            w = lambda k: self.t[k, l]  # noqa: E731
            h = rounded(plain(x, w(O.ATTN_NORM)), 1)
            q, k, v = ((h @ w(i).T).view(n, -1, d) for i in (O.WQ, O.WK, O.WV))
            q, k, v = bf16(turn(q)), self.kept(turn(k)), self.kept(v)
            o = torch.empty(n, s.n_heads, d)
            for j in range(s.n_heads):
                p = torch.softmax((q[:, j] @ k[:, j // group].T * d ** -0.5).masked_fill(later, -torch.inf), -1)
                o[:, j] = p @ v[:, j // group]
            x = x + rounded(bf16(o.reshape(n, -1)), 1) @ w(O.WO).T
            h = rounded(plain(x, w(O.MLP_NORM)), 1)
            x = x + rounded(torch.nn.functional.silu(h @ w(O.WGATE).T) * (h @ w(O.WUP).T), 1) @ w(O.WDOWN).T
        return (self.norm(x[-rows:], self.t[O.FINAL_NORM, 0]) @ self.t[O.LM_HEAD, 0].T).numpy()


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_requests_behind_one_prompt_follow_the_restatement(int8):
    rng = np.random.default_rng(3)
    base = rng.integers(0, SHAPE.vocab, 1300).tolist()
    prompts = [base + rng.integers(0, SHAPE.vocab, 3 + 5 * i).tolist() for i in range(32)]
    assert B.load().dis_k_attn_shared_in_common(32, 32, 8, 128, 1296, int8) == 1
    launches = {}
    for shared in (0, B.FLAG_ATTN_SHARED):
        e = make_engine(SHAPE, seed=5, max_batch=32, kv_pages=500, page_size=16, max_step_tokens=4096,
                        flags=B.FLAG_WEIGHTS_F8 | B.FLAG_PREFIX_CACHE | shared | (B.FLAG_KV_INT8 if int8 else 0))
        e.seq_remove(follow(e, [base], 0)[0][0])  # the base's pages are in the cache
        slots = [e.seq_add(p, InferenceParams(max_tokens=20, temperature=0.0)) for p in prompts]
        toks, _ = e.prefill(slots)
        made, logits = [[int(t)] for t in toks], []
        for _ in range(3):
            before = e.status().kernel_launches
            toks, _ = e.decode(slots)
            launches.setdefault(shared, set()).add(e.status().kernel_launches - before)
            logits.append(e.last_logits(32).copy())
            for m, t in zip(made, toks):
                m.append(int(t))
        e.close()
    (alone,), (together,) = launches[0], launches[B.FLAG_ATTN_SHARED]
    assert together - alone == 2 * (2 if int8 else 3)  # two layers: 8 bits 1 + 1 -> 1 + 3 kernels, bf16 1 -> 1 + 3
    ref = RestatedBoth(SHAPE, 5, int8)
    compared = 0
    for i in (0, 7, 18, 31):
        want = ref.logits(prompts[i] + made[i], 5)  # rows: the prompt's last, then one for each token made
        for k in range(3):
            assert rel_err(logits[k][i], want[1 + k]) <= LIMIT, (i, k)
            compared += 1
        for k, t in enumerate(made[i]):  # the greedy choice, but for near ties
            assert want[k].max() - want[k][t] <= LIMIT * np.abs(want[k]).max(), (i, k)
    assert compared == 12
