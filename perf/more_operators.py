"""Products of the decoder in 8-bit floating point whose speed and accuracy are tracked: a projection, the first layer's norm and
projection, and a whole gated feed-forward block, from one token to a prompt pass.

A case is a dict of plain values: listed() are the fixed ones, draw() gives others of the same ranges.  run() computes either the
plain form in 32-bit torch operations or, where `own` is set, makes the calls of the C ABI that a serving program makes.

Rows of activations [T][K] are held as e4m3 values with one scale per 128 entries, [ceil(K/128)][T] fp32, a power of two:
s = 2^ceil(log2(max|x| / 448)), x8 = e4m3(x / s).  Weights [N][K] have one scale per block of 128 x 128, [ceil(N/128)][ceil(K/128)] fp32,
any number; of a fused gate-up weight [2][I][K] the gate's and up's rows are blocked each by themselves.
"""
import math

import torch

own = False

# hidden size, rows of the fused qkv projection, inner size of the feed-forward block of the three Llama shapes that worker.py lists
SHAPES = {"1b": (2048, 2560, 5632), "8b": (4096, 6144, 14336), "70b": (8192, 10240, 28672)}
EPS = 1e-5


def listed():
    return [
        # attention's output of one request goes through the output projection: latency
        {"name": "linear_one", "kind": "linear", "tokens": 1, "n": 4096, "k": 4096, "out": "f32"},
        # the output projection of a decode batch
        {"name": "linear_step", "kind": "linear", "tokens": 32, "n": 8192, "k": 8192, "out": "f32"},
        # a tensor-parallel shard's odd sizes: rows that end inside a block of 128, few of them
        {"name": "linear_odd", "kind": "linear", "tokens": 77, "n": 1001, "k": 1040, "out": "bf16"},
        # the down projection of a prompt's chunk
        {"name": "linear_chunk", "kind": "linear", "tokens": 512, "n": 4096, "k": 14336, "out": "f32"},
        # the output projection of a full prompt pass
        {"name": "linear_prompt", "kind": "linear", "tokens": 6000, "n": 8192, "k": 8192, "out": "bf16"},
        # a decode step's first layer: embedding rows, norm, qkv projection
        {"name": "embed_step", "kind": "embed", "tokens": 32, "n": 6144, "k": 4096},
        # the same for a ragged prompt pass
        {"name": "embed_prompt", "kind": "embed", "tokens": 3001, "n": 6144, "k": 4096},
        # the feed-forward block of a single request: both weights are read once
        {"name": "ffn_one", "kind": "ffn", "tokens": 1, "hidden": 4096, "inner": 14336},
        # of a decode batch
        {"name": "ffn_step", "kind": "ffn", "tokens": 32, "hidden": 4096, "inner": 14336},
        # of a short prompt on the smallest shape
        {"name": "ffn_short", "kind": "ffn", "tokens": 200, "hidden": 2048, "inner": 5632},
        # sizes that fill no block
        {"name": "ffn_odd", "kind": "ffn", "tokens": 19, "hidden": 272, "inner": 720},
        # of a full prompt pass
        {"name": "ffn_prompt", "kind": "ffn", "tokens": 8192, "hidden": 4096, "inner": 14336},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "embed", "ffn", "ffn"])
    tokens = _log(rng, 1, 8192) if rng.random() < 0.7 else _log(rng, 1, 128)
    hidden, qkv, inner = SHAPES[rng.choice(["1b", "8b", "8b", "70b"])]
    if rng.random() < 0.4:  # a shard, or a model of another size
        hidden, qkv, inner = 16 * _log(rng, 4, 512), _log(rng, 16, 10240), 16 * _log(rng, 4, 1024)
    most = 2 * 8192 * 3 * 4096 * 14336
    if kind == "ffn":
        return {"kind": kind, "tokens": max(1, min(tokens, most // (6 * hidden * inner))), "hidden": hidden, "inner": inner}
    if kind == "embed":
        return {"kind": kind, "tokens": tokens, "n": qkv, "k": hidden}
    n, k = rng.choice([(hidden, hidden), (hidden, inner), (qkv, hidden)])
    return {"kind": kind, "tokens": max(1, min(tokens, most // (2 * n * k))), "n": n, "k": k, "out": rng.choice(["f32", "bf16"])}


# ------------------------------------------------------------------------------------------------ inputs
def _blocks(n):
    return -(-n // 128)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) + 1)
    return g


def _weight(g, n, k, copies=1):
    """A weight whose input channels differ in size, as trained ones' do, in 8 bits as checkpoints hold them: scale = max / 448 of a block."""
    size = (torch.rand(k, generator=g, device="cuda") + 0.5) * k ** -0.5
    w8 = torch.empty(copies * n, k, dtype=torch.float8_e4m3fn, device="cuda")
    scale = torch.empty(copies * _blocks(n), _blocks(k), device="cuda")
    for c in range(copies):
        w = torch.zeros(_blocks(n) * 128, _blocks(k) * 128, device="cuda")
        w[:n, :k] = torch.randn(n, k, generator=g, device="cuda") * size
        b = w.view(_blocks(n), 128, _blocks(k), 128)
        s = b.abs().amax((1, 3)) / 448
        w8[c * n:(c + 1) * n] = (b / s[:, None, :, None]).clamp(-448, 448).view(_blocks(n) * 128, -1)[:n, :k].to(torch.float8_e4m3fn)
        scale[c * _blocks(n):(c + 1) * _blocks(n)] = s
    return w8, scale


def _rows(g, t, k):
    """Rows of bf16 activations: tokens and channels differ in size, a few channels are far larger than the rest."""
    size = torch.rand(k, generator=g, device="cuda") + 0.5
    size[torch.randint(0, k, (max(1, k // 200),), generator=g, device="cuda")] *= 12
    return (torch.randn(t, k, generator=g, device="cuda") * size * (torch.rand(t, 1, generator=g, device="cuda") * 2 + 0.5)).to(torch.bfloat16)


def _held(s, t, k, name):
    """Where a program keeps rows of k entries in 8 bits."""
    s[name + "8"] = torch.empty(t, k, dtype=torch.uint8, device="cuda")
    s[name + "_scale"] = torch.empty(_blocks(k), t, device="cuda")


def prepare(case, seed):
    g, t, kind = _gen(seed), case["tokens"], case["kind"]
    s = {"kind": kind, "t": t}
    if kind == "ffn":
        h, i = case["hidden"], case["inner"]
        s |= {"h": h, "i": i, "x": _rows(g, t, h), "out": torch.empty(t, h, dtype=torch.bfloat16, device="cuda")}
        s["wgu8"], s["wgu_scale"] = _weight(g, i, h, 2)
        s["wd8"], s["wd_scale"] = _weight(g, h, i)
        _held(s, t, h, "x")
        _held(s, t, i, "a")
        return s
    n, k = case["n"], case["k"]
    bf16 = kind == "embed" or case["out"] == "bf16"
    s |= {"n": n, "k": k, "bf16": bf16, "out": torch.empty(t, n, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")}
    s["w8"], s["w_scale"] = _weight(g, n, k)
    _held(s, t, k, "x")
    if kind == "embed":
        vocab = 2000
        s |= {"embed": (torch.randn(vocab, k, generator=g, device="cuda") * 0.02).to(torch.bfloat16),
              "ids": torch.randint(0, vocab, (t,), generator=g, device="cuda", dtype=torch.int32),
              "gain": 1 + 0.1 * torch.randn(k, generator=g, device="cuda"), "resid": torch.empty(t, k, device="cuda")}
    else:
        s["x"] = _rows(g, t, k)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_rounded(x):
    """The values that fp32 rows stand for in 8 bits."""
    t, k = x.shape
    b = torch.nn.functional.pad(x, (0, _blocks(k) * 128 - k)).view(t, -1, 128)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True) / 448)
    s = torch.ldexp(torch.ones_like(m), e - (m == 0.5).int()).clamp_min(2.0 ** -126)
    return ((b / s).to(torch.float8_e4m3fn).float() * s).view(t, -1)[:, :k]


def _plain_weight(w8, scale):
    n, k = w8.shape
    return w8.float() * scale.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _plain(s):
    if s["kind"] == "ffn":
        i, blocks = s["i"], _blocks(s["i"])
        x = _plain_rounded(s["x"].float())
        gate = x @ _plain_weight(s["wgu8"][:i], s["wgu_scale"][:blocks]).T
        up = x @ _plain_weight(s["wgu8"][i:], s["wgu_scale"][blocks:]).T
        a = _plain_rounded(gate / (1 + (-gate).exp()) * up)
        s["out"].copy_(a @ _plain_weight(s["wd8"], s["wd_scale"]).T)
        return
    if s["kind"] == "embed":
        s["resid"].copy_(s["embed"][s["ids"].long()])
        x = s["resid"] * (s["resid"].square().mean(-1, keepdim=True) + EPS).rsqrt() * s["gain"]
    else:
        x = s["x"].float()
    s["out"].copy_(_plain_rounded(x) @ _plain_weight(s["w8"], s["w_scale"]).T)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from distributed_inference_server_b200 import binding as B
    lib, stream, t = B.load(), torch.cuda.current_stream().cuda_stream, s["t"]
    if s["kind"] == "ffn":
        rc = lib.dis_k_ffn_f8(s["x"].data_ptr(), s["wgu8"].data_ptr(), s["wgu_scale"].data_ptr(), s["wd8"].data_ptr(), s["wd_scale"].data_ptr(),
                              s["x8"].data_ptr(), s["x_scale"].data_ptr(), s["a8"].data_ptr(), s["a_scale"].data_ptr(), s["out"].data_ptr(), B.BF16, t, s["h"], s["i"], stream)
    else:
        if s["kind"] == "embed":
            rc = lib.dis_k_add_rmsnorm_f8(s["resid"].data_ptr(), s["ids"].data_ptr(), s["embed"].data_ptr(), None, 0, 0, s["gain"].data_ptr(), s["x8"].data_ptr(),
                                          s["x_scale"].data_ptr(), None, t, s["k"], EPS, stream)
        else:
            rc = lib.dis_k_quant_f8(s["x"].data_ptr(), s["x8"].data_ptr(), s["x_scale"].data_ptr(), t, s["k"], stream)
        if rc == B.OK:
            rc = lib.dis_k_gemm_f8(s["x8"].data_ptr(), s["x_scale"].data_ptr(), s["w8"].data_ptr(), s["w_scale"].data_ptr(), s["out"].data_ptr(),
                                   B.BF16 if s["bf16"] else B.F32, t, s["n"], s["k"], stream)
    if rc != B.OK:
        raise RuntimeError(lib.dis_last_error().decode())


def run(s):
    if own:
        _own(s)
    else:
        _plain(s)
    return {"x": s["resid"], "y": s["out"]} if s["kind"] == "embed" else s["out"]


# ------------------------------------------------------------------------------------------------ floors and 64-bit results
def work(case):
    t = case["tokens"]
    if case["kind"] == "ffn":
        h, i = case["hidden"], case["inner"]
        return {"bytes": 3 * h * i + 3 * 4 * _blocks(h) * _blocks(i) + 4 * t * h, "flops": 6 * t * h * i}
    n, k = case["n"], case["k"]
    rest = 2 * t * k + (2 if case["kind"] == "embed" or case["out"] == "bf16" else 4) * t * n
    if case["kind"] == "embed":
        rest += 4 * t * k + 4 * t + 4 * k
    return {"bytes": n * k + 4 * _blocks(n) * _blocks(k) + rest, "flops": 2 * t * n * k}


def _exact_rounded(x):
    """The same values from the format's definition: 3 bits behind the leading one down to 2^-6, steps of 2^-9 below, in units of the block's scale."""
    out = torch.empty_like(x)
    for k0 in range(0, x.shape[1], 128):
        b = x[:, k0:k0 + 128]
        top = b.abs().amax(1, keepdim=True)
        s = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448))), 1.0).clamp_min(2.0 ** -126)
        s = torch.where(top > 448 * s, 2 * s, torch.where((top <= 224 * s) & (s > 2.0 ** -126), s / 2, s))  # (where the logarithm was rounded)
        q = b / s
        step = torch.exp2(torch.frexp(q.abs()).exponent.double() - 4).clamp_min(2.0 ** -9)
        out[:, k0:k0 + 128] = torch.round(q / step) * step * s
    return out


def _exact_product(x, w8, scale):
    y = torch.zeros(x.shape[0], w8.shape[0], dtype=torch.float64, device=x.device)
    for r in range(0, w8.shape[0], 4096):
        w = w8[r:r + 4096].double()
        s = scale[r // 128:r // 128 + 32].double()
        w = torch.cat([w[:, c * 128:(c + 1) * 128] * torch.repeat_interleave(s[:, c], 128)[:w.shape[0], None] for c in range(scale.shape[1])], 1)
        y[:, r:r + 4096] = x @ w.T
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "ffn":
        i, b = s["i"], _blocks(s["i"])
        x = _exact_rounded(s["x"].double())
        gate, up = _exact_product(x, s["wgu8"][:i], s["wgu_scale"][:b]), _exact_product(x, s["wgu8"][i:], s["wgu_scale"][b:])
        return _exact_product(_exact_rounded(gate * torch.sigmoid(gate) * up), s["wd8"], s["wd_scale"])
    if case["kind"] == "linear":
        return _exact_product(_exact_rounded(s["x"].double()), s["w8"], s["w_scale"])
    x = s["embed"].double()[s["ids"].long()]
    n = x / (x.pow(2).sum(1, keepdim=True) / s["k"] + EPS).sqrt() * s["gain"].double()
    return {"x": x, "y": _exact_product(_exact_rounded(n), s["w8"], s["w_scale"])}
