"""Operators around the paged key/value cache whose speed and accuracy are tracked: the cache in 8 bits (written, read back, attended
over by single tokens) and attention of a batch whose requests share a long prefix, read once for all of them.

A case is a dict of plain values: listed() are the fixed ones, draw() gives others of the same ranges.  run() computes either the
plain form in 32-bit torch operations or, where `own` is set, makes the calls of the C ABI that a serving program makes.

Pages are [page][2 (K, V)][kv heads][page size][head size]; a row of the 8-bit pool (one token and kv head) stands for its whole numbers
times a scale of its own, [page][2][kv heads][page size] fp32: s = max|x| / 127, x8 = rint(x / s).
"""
import math
import random

import numpy as np
import torch

own = False

# query heads, key/value heads, head size of the three Llama shapes that worker.py lists
SHAPES = {"1b": (32, 4, 64), "8b": (32, 8, 128), "70b": (64, 8, 128)}


def listed():
    return [
        # a decode step's tokens of 32 requests join their histories (four K slices of the qkv product), the new rows are read back: latency
        {"name": "append_step", "kind": "append", "shape": "8b", "batch": 32, "new": 1, "past": 2000, "slices": 4, "whole": False, "page": 64},
        # a full prompt pass: ragged prompts join the cache, and prompt attention needs all of their histories in bf16 pages
        {"name": "append_prompt", "kind": "append", "shape": "8b", "batch": 6, "new": 2500, "past": 2048, "slices": 1, "whole": True, "page": 64},
        # the same for heads of 64 and small pages
        {"name": "append_prompt_d64", "kind": "append", "shape": "1b", "batch": 3, "new": 900, "past": 0, "slices": 1, "whole": True, "page": 16},
        # one request's history is read back for the next chunk of its prompt
        {"name": "read_one", "kind": "read", "shape": "8b", "batch": 1, "most": 1900, "page": 64},
        # sixteen long ragged histories
        {"name": "read_batch", "kind": "read", "shape": "8b", "batch": 16, "most": 6000, "page": 64},
        # decode attention of a few short requests: latency
        {"name": "decode_few", "kind": "decode", "shape": "8b", "batch": 4, "most": 500, "page": 64},
        # decode attention of a full batch whose requests have histories of very different lengths
        {"name": "decode_batch", "kind": "decode", "shape": "8b", "batch": 32, "most": 6000, "page": 64},
        # heads of 64, many requests, pages of 16
        {"name": "decode_d64", "kind": "decode", "shape": "1b", "batch": 64, "most": 3000, "page": 16},
        # two requests with very long histories, groups of eight query heads
        {"name": "decode_long", "kind": "decode", "shape": "70b", "batch": 2, "most": 60000, "page": 64},
        # eight continuations of one short prompt, heads of 64, bf16 pages
        {"name": "shared_few", "kind": "shared", "shape": "1b", "batch": 8, "prefix": 1000, "most": 100, "int8": False, "page": 64},
        # a batch behind one long system prompt, bf16 pages
        {"name": "shared_bf16", "kind": "shared", "shape": "8b", "batch": 32, "prefix": 6000, "most": 500, "int8": False, "page": 64},
        # many requests behind a longer one, 8-bit pages, groups of eight query heads
        {"name": "shared_int8", "kind": "shared", "shape": "70b", "batch": 64, "prefix": 8000, "most": 700, "int8": True, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "read", "decode", "decode", "shared", "shared"])
    shape, page = rng.choice(["1b", "8b", "8b", "70b"]), rng.choice([16, 32, 64, 64, 128])
    c = {"kind": kind, "shape": shape, "page": page}
    if kind == "append":
        if rng.random() < 0.5:
            return dict(c, batch=_log(rng, 1, 64), new=1, past=_log(rng, 16, 4000), slices=rng.choice([1, 2, 4, 8]), whole=False)
        batch = rng.randint(1, 6)
        return dict(c, batch=batch, new=_log(rng, 17, 8000 // batch if shape != "70b" else 4000 // batch), past=rng.choice([0, 0, _log(rng, 16, 2000)]), slices=1, whole=rng.random() < 0.7)
    batch = _log(rng, 1, 64)
    if kind == "read":
        return dict(c, batch=batch, most=_log(rng, 16, min(16000, 90000 // batch)))
    if kind == "decode":
        return dict(c, batch=batch, most=_log(rng, 16, min(60000, 180000 // batch)))
    return dict(c, batch=batch, prefix=_log(rng, 64, min(16000, 480000 // batch)), most=_log(rng, 1, 700), int8=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) + 1)
    return g


def _lengths(batch, most, salt=7):
    """Lengths from a few tokens to `most`, one of them `most` itself."""
    r = random.Random(salt)
    lo = math.log(max(1, most // 12))
    n = [min(most, max(1, int(math.exp(r.uniform(lo, math.log(most)))))) for _ in range(batch)]
    n[r.randrange(batch)] = most
    return n


def _tables(total, page, seed, common=0):
    """Page table [batch][most pages] of histories of `total` tokens, pages in shuffled order; the first `common` pages are the same for all."""
    pages = [-(-t // page) for t in total]
    count = common + sum(max(0, p - common) for p in pages)
    order = list(range(count))
    random.Random(int(seed) + 11).shuffle(order)
    first, at, rows = order[:common], common, []
    for p in pages:
        rows.append((first + order[at:at + p - common])[:p] + [0] * (max(pages) - p))
        at += max(0, p - common)
    return count, torch.tensor(rows, dtype=torch.int32, device="cuda")


def _quantise(x):
    """Rows of x (last dimension) in 8 bits: whole numbers and the row's scale."""
    s = x.abs().amax(-1) / 127
    return torch.round(x / torch.where(s > 0, s, 1.0)[..., None]), s


def _cache(g, pages, page, nkv, d, int8):
    """A pool of keys and values whose rows differ in size and whose key channels do, as trained models' do."""
    size = torch.rand(2, nkv, 1, d, generator=g, device="cuda") + 0.5
    x = torch.randn(pages, 2, nkv, page, d, generator=g, device="cuda") * size * (torch.rand(pages, 2, nkv, page, 1, generator=g, device="cuda") + 0.5)
    if not int8:
        return x.to(torch.bfloat16), None
    q, s = _quantise(x)
    return q.to(torch.int8), s


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    nh, nkv, d = SHAPES[case["shape"]]
    g, page, batch, kind = _gen(seed), case["page"], case["batch"], case["kind"]
    s = {"kind": kind, "nh": nh, "nkv": nkv, "d": d, "page": page, "batch": batch}
    if kind == "append":
        new = _lengths(batch, case["new"])
        past = _lengths(batch, case["past"], 9) if case["past"] else [0] * batch
        total = [a + b for a, b in zip(new, past)]
        T = sum(new)
        pos = torch.cat([torch.arange(a, a + b) for a, b in zip(past, new)]).int().cuda()
        freq = 500000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        angle = torch.arange(max(total), device="cuda", dtype=torch.float64)[:, None] * freq
        s |= {"T": T, "slices": case["slices"], "pos": pos, "row": torch.repeat_interleave(torch.arange(batch), torch.tensor(new)).int().cuda(),
              "cos": angle.cos().float(), "sin": angle.sin().float(), "qkv": torch.randn(case["slices"], T, (nh + 2 * nkv) * d, generator=g, device="cuda") * case["slices"] ** -0.5,
              "q": torch.zeros(T, nh * d, dtype=torch.bfloat16, device="cuda"), "first": _int32([0] * batch if case["whole"] else past)}
        int8 = True
    elif kind == "read":
        total, int8 = _lengths(batch, case["most"]), True
        s["first"] = _int32([0] * batch)
    else:
        prefix = case.get("prefix", 0)
        total, int8 = [prefix + n for n in _lengths(batch, case["most"])], case.get("int8", True)
        s |= {"prefix": prefix, "q": (torch.randn(batch, nh * d, generator=g, device="cuda") * 1.5).to(torch.bfloat16),
              "out": torch.zeros(batch, nh * d, dtype=torch.bfloat16, device="cuda")}
    # whole pages of the prefix are shared; where it ends inside a page, every request has a copy of that page's part
    pages, s["table"] = _tables(total, page, seed, case.get("prefix", 0) // page)
    s["pool"], s["scale"] = _cache(g, pages, page, nkv, d, int8)
    s["pages"], s["ctx"], s["rows"], s["most"] = pages, _int32(total), torch.arange(batch, dtype=torch.int32, device="cuda"), max(total)
    if case.get("prefix", 0) % page:
        at = case["prefix"] // page
        part, own_pages = case["prefix"] % page, s["table"][:, at].long()
        s["pool"][own_pages, :, :, :part] = s["pool"][own_pages[:1], :, :, :part]
        if int8:
            s["scale"][own_pages, :, :, :part] = s["scale"][own_pages[:1], :, :, :part]
    if kind in ("append", "read"):
        s["read"] = torch.zeros(pages, 2, nkv, page, d, dtype=torch.bfloat16, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_write(s):
    T, nh, nkv, d, page = s["T"], s["nh"], s["nkv"], s["d"], s["page"]
    x = s["qkv"].sum(0).view(T, nh + 2 * nkv, d)
    pos, row = s["pos"].long(), s["row"].long()
    c, n = s["cos"][pos][:, None], s["sin"][pos][:, None]
    a, b = x[:, :nh + nkv, :d // 2], x[:, :nh + nkv, d // 2:]
    rot = torch.cat([a * c - b * n, b * c + a * n], -1)
    s["q"].copy_(rot[:, :nh].reshape(T, nh * d))
    kv, scale = _quantise(torch.stack([rot[:, nh:], x[:, nh + nkv:]], 1))
    at = s["table"][row, pos // page].long()
    s["pool"][at, :, :, pos % page] = kv.to(torch.int8)
    s["scale"][at, :, :, pos % page] = scale


def _plain_read(s):
    page = s["page"]
    pos = torch.arange(s["most"], device="cuda").expand(s["batch"], -1)
    row, pos = ((pos >= s["first"][:, None]) & (pos < s["ctx"][:, None])).nonzero(as_tuple=True)
    at, slot = s["table"][row, pos // page].long(), pos % page
    s["read"][at, :, :, slot] = (s["pool"][at, :, :, slot].float() * s["scale"][at, :, :, slot][..., None]).to(torch.bfloat16)


def _plain_attention(s):
    B, nh, nkv, d = s["batch"], s["nh"], s["nkv"], s["d"]
    table = s["table"].long()
    kv = s["pool"][table].float()  # [batch][pages][2][kv heads][page][d]
    if s["scale"] is not None:
        kv = kv * s["scale"][table][..., None]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, B, nkv, -1, d)
    w = s["q"].float().view(B, nkv, nh // nkv, d) @ kv[0].transpose(-1, -2) * d ** -0.5
    w = w.masked_fill(torch.arange(kv.shape[3], device="cuda") >= s["ctx"][:, None, None, None], -math.inf)
    w = (w - w.amax(-1, keepdim=True)).exp()
    s["out"].copy_((w @ kv[1] / w.sum(-1, keepdim=True)).reshape(B, nh * d))


# ------------------------------------------------------------------------------------------------ the framework's calls
_kept = {}


def _workspace(lib, floats):
    """What a server keeps for all of its calls: zero once, left so by every call."""
    if _kept.get("floats", 0) < floats:
        _kept["floats"], _kept["area"] = floats, torch.zeros(floats, dtype=torch.float32, device="cuda")
    return _kept["area"].data_ptr()


def _own(s):
    from distributed_inference_server_b200 import binding as B
    lib, stream, kind = B.load(), torch.cuda.current_stream().cuda_stream, s["kind"]
    nh, nkv, d, page, width = s["nh"], s["nkv"], s["d"], s["page"], s["table"].shape[1]
    rc = B.OK
    if kind == "append":
        rc = lib.dis_k_rope_kv_write_i8(s["qkv"].data_ptr(), s["slices"], s["qkv"].stride(0), s["q"].data_ptr(), s["pool"].data_ptr(), s["scale"].data_ptr(),
                                        s["table"].data_ptr(), width, s["row"].data_ptr(), s["pos"].data_ptr(), s["cos"].data_ptr(), s["sin"].data_ptr(),
                                        s["T"], nh, nkv, d, page, stream)
    if kind in ("append", "read") and rc == B.OK:
        rc = lib.dis_k_kv_read_i8(s["pool"].data_ptr(), s["scale"].data_ptr(), s["read"].data_ptr(), s["table"].data_ptr(), s["table"].data_ptr(), width,
                                  s["rows"].data_ptr(), s["first"].data_ptr(), s["ctx"].data_ptr(), s["batch"], nkv, d, page, stream)
    if kind == "decode":
        area = _workspace(lib, lib.dis_k_attn_paged_i8_scratch_elems(s["batch"], nh, nkv, d))
        rc = lib.dis_k_attn_paged_i8(s["q"].data_ptr(), s["pool"].data_ptr(), s["scale"].data_ptr(), s["table"].data_ptr(), width, s["rows"].data_ptr(),
                                     s["ctx"].data_ptr(), s["out"].data_ptr(), area, s["batch"], nh, nkv, d, page, stream)
    if kind == "shared":
        area = _workspace(lib, lib.dis_k_attn_shared_scratch_elems(s["batch"], nh, nkv, d))
        rc = lib.dis_k_attn_shared(s["q"].data_ptr(), s["pool"].data_ptr(), s["scale"].data_ptr() if s["scale"] is not None else None, s["pages"],
                                   s["table"].data_ptr(), width, s["rows"].data_ptr(), s["ctx"].data_ptr(), s["prefix"], s["out"].data_ptr(), area,
                                   s["batch"], nh, nkv, d, page, stream)
    if rc != B.OK:
        raise RuntimeError(lib.dis_last_error().decode())


def run(s):
    if own:
        _own(s)
    elif s["kind"] == "append":
        _plain_write(s)
        _plain_read(s)
    elif s["kind"] == "read":
        _plain_read(s)
    else:
        _plain_attention(s)
    if s["kind"] == "append":
        return {"q": s["q"], "read": s["read"]}
    return s["read"] if s["kind"] == "read" else s["out"]


# ------------------------------------------------------------------------------------------------ floors and 64-bit results
def work(case):
    nh, nkv, d = SHAPES[case["shape"]]
    row = 2 * nkv * (d + 4)  # a token's keys and values in 8 bits
    if case["kind"] == "append":
        new = sum(_lengths(case["batch"], case["new"]))
        past = sum(_lengths(case["batch"], case["past"], 9)) if case["past"] else 0
        read = new + (past if case["whole"] else 0)
        kept = row * (read - new)  # what was written a moment ago need not come from memory again
        return {"bytes": new * (case["slices"] * (nh + 2 * nkv) * d * 4 + nh * d * 2 + row + d * 4) + kept + read * 4 * nkv * d,
                "flops": new * (nh + 2 * nkv) * d * (case["slices"] + 4)}
    if case["kind"] == "read":
        n = sum(_lengths(case["batch"], case["most"]))
        return {"bytes": n * (row + 4 * nkv * d), "flops": n * 2 * nkv * d}
    n = sum(_lengths(case["batch"], case["most"]))
    prefix = case.get("prefix", 0)
    row = row if case.get("int8", True) else 4 * nkv * d
    return {"bytes": (n + prefix) * row + case["batch"] * 4 * nh * d, "flops": 4 * nh * d * (n + case["batch"] * prefix)}


def exact(case, seed):
    s = prepare(case, seed)
    nh, nkv, d, page, batch = s["nh"], s["nkv"], s["d"], s["page"], s["batch"]
    value = lambda p: s["pool"][p].double() * (1.0 if s["scale"] is None else s["scale"][p].double()[..., None])  # noqa: E731
    if case["kind"] in ("decode", "shared"):
        out = torch.empty(batch, nh, d, dtype=torch.float64, device="cuda")
        for b in range(batch):
            n = int(s["ctx"][b])
            kv = value(s["table"][b, :-(-n // page)].long())
            for h in range(nkv):
                k, v = kv[:, 0, h].reshape(-1, d)[:n], kv[:, 1, h].reshape(-1, d)[:n]
                heads = slice(h * (nh // nkv), (h + 1) * (nh // nkv))
                out[b, heads] = torch.softmax(s["q"].double().view(batch, nh, d)[b, heads] @ k.T / math.sqrt(d), -1) @ v
        return out.view(batch, nh * d)
    read = torch.zeros(s["read"].shape, dtype=torch.float64, device="cuda")
    for b in range(batch):
        lo, hi = int(s["first"][b]), int(s["ctx"][b])
        for p in range(lo // page, -(-hi // page)):
            at, a, e = int(s["table"][b, p]), max(lo - p * page, 0), min(hi - p * page, page)
            read[at, :, :, a:e] = value(at)[:, :, a:e]
    if case["kind"] == "read":
        return read
    x = s["qkv"].double().sum(0).view(-1, nh + 2 * nkv, d)
    z = torch.view_as_complex(torch.stack([x[:, :nh + nkv, :d // 2], x[:, :nh + nkv, d // 2:]], -1).contiguous())
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
    rot = torch.cat([(z * turn).real, (z * turn).imag], -1)
    kv = torch.stack([rot[:, nh:], x[:, nh + nkv:]], 1)
    unit = kv.abs().amax(-1, keepdim=True) / 127
    read[s["table"][s["row"].long(), s["pos"].long() // page].long(), :, :, s["pos"].long() % page] = torch.round(kv / unit) * unit
    return {"q": rot[:, :nh].reshape(-1, nh * d), "read": read}
