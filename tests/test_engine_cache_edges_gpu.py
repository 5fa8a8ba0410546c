"""Engines with DIS_FLAG_KV_INT8 and DIS_FLAG_ATTN_SHARED in the ways that tests/test_engine_cache_gpu.py does not take."""
import numpy as np
import pytest

from distributed_inference_server_b200 import binding as B
from tests.test_engine_cache_gpu import SMALL, follow
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
