"""Engines with DIS_FLAG_KV_INT8 and DIS_FLAG_ATTN_SHARED in the ways that tests/test_engine_cache_gpu.py does not take: through the continuous batcher, with
too few sequences to share, with classes of kernels left out."""
import numpy as np
import pytest

from distributed_inference_server_b200 import ContinuousBatcher, InferenceParams
from distributed_inference_server_b200 import binding as B
from oracle import oracle as O
from tests.test_engine_cache_gpu import SMALL, TOL, follow
from tests.test_engine_gpu import make_engine

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("skip", ["rope", "attn"])
def test_classes_left_out_of_an_int8_step(monkeypatch, skip):
    """DIS_DEBUG_SKIP (measurement: results are garbage) leaves the write and the attention out of steps over 8-bit pages, as of the others."""
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, SMALL.vocab, n).tolist() for n in (40, 70)]
    runs = []
    for env in (None, None, skip):
        if env:
            monkeypatch.setenv("DIS_DEBUG_SKIP", env)
        e = make_engine(SMALL, seed=7, flags=B.FLAG_KV_INT8)
        runs.append(follow(e, prompts, 1)[2][0])
        e.close()
    assert np.array_equal(runs[0], runs[1]) and not np.array_equal(runs[0], runs[2])


LONG = O.ModelShape(1024, 256, 2, 32, 8, 128, 704, 2048)


def behind(base, n, rng):
    return [base + [i] + rng.integers(0, LONG.vocab, 3 + 2 * i).tolist() for i in range(n)]


@pytest.mark.parametrize("int8", [0, B.FLAG_KV_INT8], ids=["bf16", "int8"])
def test_two_sequences_are_too_few_to_share(int8):
    """Steps of two sequences behind a common prompt: the launches of an engine without the flag, and its logits to the bit."""
    rng = np.random.default_rng(8)
    base = rng.integers(0, LONG.vocab, 1776).tolist()
    prompts = behind(base, 2, rng)
    assert B.load().dis_k_attn_shared_in_common(2, 32, 8, 128, 1776, int8 != 0) == 0
    runs = []
    for shared in (0, B.FLAG_ATTN_SHARED):
        e = make_engine(LONG, seed=5, max_batch=8, kv_pages=400, page_size=16, max_step_tokens=4096, flags=B.FLAG_PREFIX_CACHE | shared | int8)
        e.seq_remove(follow(e, [base], 0)[0][0])
        slots = [e.seq_add(p, InferenceParams(max_tokens=8, temperature=0.0)) for p in prompts]
        e.prefill(slots)
        run = []
        for _ in range(3):
            before = e.status().kernel_launches
            e.decode(slots)
            run.append((e.status().kernel_launches - before, e.last_logits(2).copy()))
        runs.append(run)
        e.close()
    for (n0, a), (n1, b) in zip(*runs):
        assert n0 == n1 and np.array_equal(a, b)


@pytest.mark.parametrize("int8", [0, B.FLAG_KV_INT8], ids=["bf16", "int8"])
def test_batcher_with_common_pages(int8):
    """Requests behind one prompt through the continuous batcher, prompts read beside running sequences: every request gets the tokens that an engine without
    the shared flag gives it, but for near ties, and steps of running sequences launch the shared attention."""
    rng = np.random.default_rng(9)
    base = rng.integers(0, LONG.vocab, 1776).tolist()
    prompts, new = behind(base, 24, rng), 6
    assert B.load().dis_k_attn_shared_in_common(24, 32, 8, 128, 1776, int8 != 0) == 1
    kw = dict(seed=5, max_batch=24, kv_pages=500, page_size=16, max_step_tokens=2048)
    e = make_engine(LONG, flags=B.FLAG_PREFIX_CACHE | int8, **kw)
    e.seq_remove(follow(e, [base], 0)[0][0])
    slots = [e.seq_add(p, InferenceParams(max_tokens=new, temperature=0.0)) for p in prompts]
    toks, _ = e.prefill(slots)
    rows, want = [e.last_logits(24).copy()], [[int(t)] for t in toks]
    for _ in range(new - 1):
        before = e.status().kernel_launches
        toks, _ = e.decode(slots)
        plain = e.status().kernel_launches - before
        rows.append(e.last_logits(24).copy())
        for w, t in zip(want, toks):
            w.append(int(t))
    e.close()
    e = make_engine(LONG, flags=B.FLAG_PREFIX_CACHE | B.FLAG_ATTN_SHARED | int8, **kw)
    e.seq_remove(follow(e, [base], 0)[0][0])
    cb = ContinuousBatcher(e, max_active=24)
    cb.set_prefill_budget(300)  # prompts' tails are read over several passes, beside sequences that run already
    for i, p in enumerate(prompts):
        cb.submit(i, p, InferenceParams(new, 0.0))
    got, launches = {i: [] for i in range(24)}, []
    for _ in range(200):
        before = e.status().kernel_launches
        events = cb.step()
        launches.append(e.status().kernel_launches - before)
        for ev in events:
            if ev[1] == B.EVENT_TOKEN:
                got[ev[0]].append(ev[2])
        d = cb.depth()
        if d.total == 0 and d.active == 0 and not events:
            break
    assert plain + (4 if int8 else 6) in launches, (plain, launches)  # two layers: write and attention, or one kernel, became four
    for i in range(24):
        assert len(got[i]) == new
        for k in range(new):
            if got[i][k] != want[i][k]:  # a near tie: the histories differ from here on
                row = rows[k][i]
                assert row.max() - row[got[i][k]] <= TOL * np.abs(row).max(), (i, k)
                break
    cb.close()
    e.close()
