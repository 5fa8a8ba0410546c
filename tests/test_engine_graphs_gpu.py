"""CUDA graphs of decode steps: one per launch of the step, whatever the length of a common prefix or of the histories is, and a bounded number of them."""
import numpy as np
import pytest

from distributed_inference_server_b200 import InferenceParams
from distributed_inference_server_b200 import binding as B
from oracle import oracle as O
from tests.test_engine_gpu import make_engine, rel_err

pytestmark = pytest.mark.gpu
TOL = 2e-2  # of max|logit|, as in the other engine tests


@pytest.mark.parametrize("int8", [0, B.FLAG_KV_INT8], ids=["bf16", "int8"])
def test_one_graph_serves_common_prefixes_of_many_lengths(int8):
    """Twenty lengths, 153 key tiles to 145 and as many slices each: one graph, captured at the longest prefix, and the logits of an engine that reads
    every history by itself."""
    shape = O.ModelShape(512, 256, 2, 32, 8, 128, 320, 10240)
    rng = np.random.default_rng(11)
    lengths = [9792 - 16 * k for k in range(0, 33, 2)] + [9280 + 16 * k for k in (1, 3, 5)]
    base = rng.integers(0, shape.vocab, 9792).tolist()
    tails = [[rng.integers(0, shape.vocab, 3 + i).tolist() for i in range(16)] for _ in lengths]
    runs = []
    for shared in (0, B.FLAG_ATTN_SHARED):
        e = make_engine(shape, seed=5, max_batch=16, kv_pages=2000, page_size=16, max_step_tokens=10240, flags=B.FLAG_PREFIX_CACHE | shared | int8)
        P = InferenceParams(max_tokens=4, temperature=0.0)
        s = e.seq_add(base + [1], P)
        e.prefill([s])
        e.seq_remove(s)
        logits = []
        for n, tail in zip(lengths, tails):
            assert B.load().dis_k_attn_shared_in_common(16, 32, 8, 128, n, int8 != 0) == 1
            slots = [e.seq_add(base[:n] + [i] + t, P) for i, t in enumerate(tail)]  # (each tail begins with another token: nothing more is common)
            first, _ = e.prefill(slots)
            before = e.status().kernel_launches
            e.decode(slots)
            logits.append((e.last_logits(16).copy(), first.copy(), e.status().kernel_launches - before))
            for s in slots:
                e.seq_remove(s)
        runs.append((logits, e.graph_stats()))
        e.close()
    assert {b[2] - a[2] for a, b in zip(runs[0][0], runs[1][0])} == {4}  # every length was read once: two kernels a layer became four
    assert runs[1][1] == (1, 1), runs[1][1]
    for n, a, b in zip(lengths, runs[0][0], runs[1][0]):
        same = a[1] == b[1]  # (prompts run alike in both engines)
        assert bool(same.all())
        assert rel_err(b[0], a[0]) <= TOL, n


def test_int8_engine_keeps_its_graph_as_histories_grow():
    shape = O.ModelShape(512, 256, 2, 8, 2, 128, 320, 8192)
    rng = np.random.default_rng(12)
    e = make_engine(shape, seed=5, max_batch=4, kv_pages=1200, page_size=16, max_step_tokens=8192, flags=B.FLAG_KV_INT8)
    P = InferenceParams(max_tokens=4, temperature=0.0)
    for n in (20, 300, 900, 2500, 8000):
        slots = [e.seq_add(rng.integers(0, shape.vocab, max(5, n // (i + 1))).tolist(), P) for i in range(4)]
        e.prefill(slots)
        e.decode(slots)
        for s in slots:
            e.seq_remove(s)
    assert e.graph_stats() == (1, 1)
    e.close()


def test_graphs_are_bounded(monkeypatch):
    """With room for three: six batch sizes twice over, the same logits as with room for all, never more than three kept."""
    shape = O.ModelShape(512, 256, 2, 8, 2, 64, 320, 512)
    rng = np.random.default_rng(13)
    prompts = [rng.integers(0, shape.vocab, 10 + 7 * i).tolist() for i in range(6)]
    runs = []
    for most in (None, "3"):
        if most:
            monkeypatch.setenv("DIS_MAX_GRAPHS", most)
        e = make_engine(shape, seed=6, max_batch=8, kv_pages=100, page_size=16)
        P = InferenceParams(max_tokens=40, temperature=0.0)
        slots = [e.seq_add(p, P) for p in prompts]
        e.prefill(slots)
        out, stats = [], []
        for n in (1, 2, 3, 4, 5, 6) * 2:
            e.decode(slots[:n])
            out.append(e.last_logits(n).copy())
            stats.append(e.graph_stats())
        if most:
            assert e.replay_last_step(2) > 0.0
        runs.append((out, stats))
        e.close()
    assert runs[0][1][-1] == (6, 6)
    assert max(k for k, _ in runs[1][1]) == 3 and runs[1][1][-1][1] == 12
    for a, b in zip(runs[0][0], runs[1][0]):
        assert np.array_equal(a, b)
