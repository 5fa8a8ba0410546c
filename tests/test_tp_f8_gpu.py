"""Tensor-parallel engines with their projections in 8-bit floating point (DIS_FLAG_WEIGHTS_F8), a rank at a time on one GPU.

A rank runs by itself, in a process of its own, beside a stand-in for the collectives that waits for nobody: its all-reduce returns the rank's own
contribution, its all-gather the rank's own part in every rank's place.  What the rank then computes is a decoder of its own heads and inner entries alone, which
the restatement of test_engine_f8_gpu.py computes from the slices of shard_plan.py.  (The exchange over peer memory needs the other ranks.)"""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from distributed_inference_server_b200 import binding as B
from distributed_inference_server_b200 import shard_plan as SP
from oracle import oracle as O
from tests.test_engine_cache_gpu import Restated, bf16
from tests.test_engine_f8_gpu import RestatedF8, bits, rounded, tol
from tests.test_engine_gpu import rel_err

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHAPE = O.ModelShape(1024, 256, 3, 8, 4, 64, 768, 512)     # every rank's part starts on a block of 128
RAGGED = O.ModelShape(1024, 272, 2, 8, 4, 64, 704, 512)    # inner parts of 352 rows: they start inside one
PROJECTIONS = (O.WQ, O.WK, O.WV, O.WO, O.WGATE, O.WUP, O.WDOWN)

STAND_IN = r"""
#include <dlfcn.h>
#include <stddef.h>
typedef struct { char bytes[128]; } id_t_;
typedef int (*copy_t)(unsigned long long, unsigned long long, size_t, void *);
static int ranks;
static int copy(const void *from, void *to, size_t n, void *stream) {
  static copy_t f;
  if (!f) f = (copy_t)dlsym(dlopen("libcuda.so.1", RTLD_NOW), "cuMemcpyDtoDAsync_v2");
  return from == to ? 0 : f((unsigned long long)to, (unsigned long long)from, n, stream);
}
int ncclGetUniqueId(id_t_ *id) { return 0; }
int ncclCommInitRank(void **comm, int n, id_t_ id, int rank) { ranks = n; *comm = &ranks; return 0; }
int ncclCommDestroy(void *comm) { return 0; }
int ncclAllReduce(const void *s, void *r, size_t n, int type, int op, void *comm, void *stream) { return copy(s, r, n * 4, stream); }
int ncclAllGather(const void *s, void *r, size_t n, int type, void *comm, void *stream) {
  for (int i = 0; i < ranks; i++) { int e = copy(s, (char *)r + i * n * 4, n * 4, stream); if (e) return e; }
  return 0;
}
const char *ncclGetErrorString(int e) { return "stand-in"; }
"""

RANK = r"""
import ctypes, json, sys
import numpy as np
job = json.load(open(sys.argv[1]))
ctypes.CDLL(job["lib"], ctypes.RTLD_GLOBAL)
from distributed_inference_server_b200 import Engine, InferenceParams, ModelShape, WorkerConfig, WorkerError
from distributed_inference_server_b200 import binding as B
e = Engine(WorkerConfig(ModelShape(*job["shape"]), tp_rank=job["rank"], tp_size=2, max_batch=8, kv_pages=64, page_size=16, max_step_tokens=256, nccl_id=bytes(128),
                        flags=job["flags"]))
out, said = {}, ""
if job["how"] == "synthetic":
    e.load_synthetic(job["seed"])
else:
    t = np.load(job["tensors"])
    for name in t.files:
        what, kind, layer = name.split("_")
        if what == "plain":
            e.load_tensor(int(kind), int(layer), t[name])
        elif what == "bytes":
            try:
                e.load_tensor_f8(int(kind), int(layer), t[name], t[f"scales_{kind}_{layer}"])
            except WorkerError as err:
                said += f"{kind}: {err}\n"
    out["said"] = np.array(said)
if not said:
    e.finalize()
    slots = [e.seq_add(p, InferenceParams(max_tokens=8, temperature=0.0)) for p in job["prompts"]]
    toks, _ = e.prefill(slots)
    made = [[int(x)] for x in toks]
    for i in range(4):
        toks, _ = e.decode(slots)
        out[f"logits_{i}"] = e.last_logits(len(slots))
        for m, x in zip(made, toks):
            m.append(int(x))
    out["made"] = np.array(made)
    for kind in job["kinds"]:
        for layer in range(job["shape"][2]):
            out[f"read_{kind}_{layer}"] = e.read_tensor(kind, layer)
np.savez(job["out"], **out)
e.close()
"""


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    d = tmp_path_factory.mktemp("nccl")
    (d / "nccl.c").write_text(STAND_IN)
    (d / "rank.py").write_text(RANK)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-Wl,-soname,libnccl.so.2", str(d / "nccl.c"), "-o", str(d / "libnccl.so.2"), "-ldl"], check=True)
    return d


def run_rank(d, shape, rank, how, prompts, tensors=None, flags=0):
    job = {"lib": str(d / "libnccl.so.2"), "shape": [shape.vocab, shape.hidden, shape.layers, shape.n_heads, shape.n_kv_heads, shape.head_dim, shape.inter, shape.max_ctx,
           shape.rope_theta, shape.rms_eps], "rank": rank, "how": how, "seed": 7, "flags": flags | B.FLAG_WEIGHTS_F8, "prompts": prompts, "kinds": list(PROJECTIONS),
           "out": str(d / "out.npz"), "tensors": str(d / "tensors.npz")}
    if tensors:
        np.savez(job["tensors"], **tensors)
    (d / "job.json").write_text(json.dumps(job))
    r = subprocess.run([sys.executable, str(d / "rank.py"), str(d / "job.json")], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return np.load(job["out"])


class RankAlone(RestatedF8):
    """The restatement of one rank's heads and inner entries."""

    def __init__(self, shape, weights, rank):
        self.s = O.ModelShape(shape.vocab // 2, shape.hidden, shape.layers, shape.n_heads // 2, shape.n_kv_heads // 2, shape.head_dim, shape.inter // 2, shape.max_ctx,
                              shape.rope_theta, shape.rms_eps)
        self.t = {}
        for (k, l), a in weights.items():
            rows, cols = SP.shard_slices(shape, k, rank, 2)
            self.t[k, l] = a[rows, cols].contiguous() if a.ndim == 2 else a


def follows(out, ref, prompts, shape, rank):
    half = shape.vocab // 2
    for i, p in enumerate(prompts):
        made = out["made"][i].tolist()
        want = ref.logits(p + made)
        for k in range(4):
            got = out[f"logits_{k}"][i]
            assert np.array_equal(got[:half], got[half:])  # (the rank's own part twice)
            assert rel_err(got[:half], want[len(p) + k]) <= tol(shape), (i, k)
        for k, x in enumerate(made):
            row = want[len(p) - 1 + k]
            assert row.max() - row[x - rank * half] <= tol(shape) * np.abs(row).max()  # the rank's greedy choice, but for near ties


def prompts_of(shape):
    rng = np.random.default_rng(3)
    return [rng.integers(0, shape.vocab, n).tolist() for n in (5, 40, 180)]  # (prompts together: products in pairs; decode: in tiles)


@pytest.mark.parametrize("rank", [0, 1])
@pytest.mark.parametrize("shape", [SHAPE, RAGGED], ids=["blocks", "ragged"])
def test_a_ranks_part_of_bf16_tensors(stand_in, shape, rank):
    """Generated in bf16, sliced, turned into 8 bits in blocks that start where the slice does."""
    prompts = prompts_of(shape)
    out = run_rank(stand_in, shape, rank, "synthetic", prompts)
    ref = RankAlone(shape, Restated(shape, 7).t, rank)
    for (k, l), a in ref.t.items():
        if k in PROJECTIONS:
            ref.t[k, l] = rounded(bf16(a), 2)
            assert np.array_equal(out[f"read_{k}_{l}"], bits(ref.t[k, l]).reshape(-1)), (k, l)
    follows(out, ref, prompts, shape, rank)


def eight_bit_tensors(shape):
    """(arrays for the rank's process, {(kind, layer): values}) of a checkpoint in 8 bits with scales of its own, other tensors in fp32"""
    arrays, values = {}, {}
    for (k, l), a in Restated(shape, 7).t.items():
        if k not in PROJECTIONS:
            arrays[f"plain_{k}_{l}"], values[k, l] = a.numpy(), a
            continue
        n, m = a.shape
        pad = torch.nn.functional.pad(a, (0, -m % 128, 0, -n % 128))
        b = pad.view(-1, 128, pad.shape[1] // 128, 128)
        s = b.abs().amax((1, 3)) / 448
        q = (b / s[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        arrays[f"bytes_{k}_{l}"] = q.view(pad.shape)[:n, :m].contiguous().view(torch.uint8).numpy()
        arrays[f"scales_{k}_{l}"] = s.numpy()
        values[k, l] = (q.float() * s[:, None, :, None]).view(pad.shape)[:n, :m].contiguous()
    return arrays, values


@pytest.mark.parametrize("rank", [0, 1])
def test_a_ranks_part_of_tensors_in_8_bits(stand_in, rank):
    prompts = prompts_of(SHAPE)
    arrays, values = eight_bit_tensors(SHAPE)
    out = run_rank(stand_in, SHAPE, rank, "loaded", prompts, arrays)
    assert str(out["said"]) == ""
    ref = RankAlone(SHAPE, values, rank)
    for (k, l), a in ref.t.items():
        if k in PROJECTIONS:
            assert np.array_equal(out[f"read_{k}_{l}"], bits(a).reshape(-1)), (k, l)
    follows(out, ref, prompts, SHAPE, rank)


def test_a_part_that_starts_inside_a_block_is_refused(stand_in):
    arrays, _ = eight_bit_tensors(RAGGED)
    said = str(run_rank(stand_in, RAGGED, 1, "loaded", [], arrays)["said"]).splitlines()
    assert {int(s.split(":")[0]) for s in said} == {O.WGATE, O.WUP, O.WDOWN} and all("inside a block of 128" in s for s in said)


def test_ranks_whose_heads_fill_no_block_are_refused(stand_in):
    with pytest.raises(AssertionError) as err:  # 2 kv heads of 64 over two ranks
        run_rank(stand_in, O.ModelShape(1024, 256, 1, 8, 2, 64, 768, 512), 0, "synthetic", [])
    assert "multiples of 128" in str(err.value)
