"""The paged cache's operators, as cases with a size each, in their plain form and through the framework's calls.

A serving program keeps the keys and values of many sequences as codes in the pages of one pool. Three operators work on it:

* append: a step's new tokens. Keys (and queries) are normed per head and rotated to their positions, keys and values are
  quantised, and the codes and scales go to the tokens' slots of the pool; the rotated queries come back in their own type.
* read: ranges of the sequences' tokens, found through the page tables, come back as vectors (for a chunk of a prompt
  that attends with a kernel of its own, or to move a prefix).
* attend: one new token of every sequence attends over the sequence's pages, read as codes, with capped scores, a bias by
  distance or a sliding window where the model has them.

Fields of a case: kv and queries (KV heads, query heads per KV head), dim, kmethod / kbits and vmethod / vbits (the codes),
page (tokens), layout ("head": [page][head][slot], "token": [page][slot][head]), dtype (of the vectors). append: tokens, norm,
rotary (rotated coordinates, 0 for none), padded (tokens of the batch that are padding, with slot -1). read and attend:
sequences, tokens (the longest), ragged (lengths spread from one token up), empty (sequences of length zero at the end).
attend: softcap, window, slopes.

Codes are compared as the packed bytes that the pool holds: whole numbers. Sizes are those of pitch_amd/workloads.py and
bench.py (GPT-2-small: 12 heads of 64; Qwen2.5-1.5B: 2 KV heads of 128 under 12 query heads; Llama-3-8B: 8 KV heads of 128
under 32 query heads), with batches and lengths of ordinary and ragged sizes.
"""
from __future__ import annotations

import json
import math
from pathlib import Path

import numpy as np
import torch

own = False
DEVICE = "cuda"
SEED = 0x50495443
EPS = 1e-6
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed() -> list[dict]:
    return [
        # one sequence's new token of a Llama-3-8B-sized layer with normed queries and keys: the smallest step
        dict(name="append_one_bf16", kind="append", tokens=1, padded=0, kv=8, queries=4, dim=128, kmethod="turboQuant", kbits=4,
             vmethod="turboQuant", vbits=4, page=16, layout="head", norm=True, rotary=128, dtype="bfloat16"),
        # a decode step of 48 sequences in a batch padded to 64, keys of four bits and values of three
        dict(name="append_step_bf16", kind="append", tokens=64, padded=16, kv=8, queries=4, dim=128, kmethod="turboQuant",
             kbits=4, vmethod="turboQuant", vbits=3, page=64, layout="head", norm=True, rotary=128, dtype="bfloat16"),
        # a prompt of 8191 tokens of the same layer
        dict(name="append_prompt_bf16", kind="append", tokens=8191, padded=0, kv=8, queries=4, dim=128, kmethod="turboQuant",
             kbits=4, vmethod="turboQuant", vbits=4, page=64, layout="head", norm=True, rotary=128, dtype="bfloat16"),
        # a chunk of 2001 tokens of a Qwen2.5-1.5B layer, PolarQuant, half of the coordinates rotated, token-major pages
        dict(name="append_polar_f16", kind="append", tokens=2001, padded=0, kv=2, queries=6, dim=128, kmethod="polarQuant",
             kbits=4, vmethod="polarQuant", vbits=3, page=32, layout="token", norm=False, rotary=64, dtype="float16"),
        # one sequence's first 77 tokens read back for a chunk of its prompt
        dict(name="read_short_bf16", kind="read", sequences=1, tokens=77, ragged=False, empty=0, kv=8, dim=128,
             kmethod="turboQuant", kbits=4, vmethod="turboQuant", vbits=4, page=16, layout="head", dtype="bfloat16"),
        # the prefixes of 16 sequences of up to 4000 tokens, eight KV heads
        dict(name="read_prefixes_bf16", kind="read", sequences=16, tokens=4000, ragged=True, empty=1, kv=8, dim=128,
             kmethod="turboQuant", kbits=4, vmethod="turboQuant", vbits=3, page=64, layout="head", dtype="bfloat16"),
        # a GPT-2 layer at 32767 tokens in float32, heads of 64, pages of 48 tokens
        dict(name="read_gpt2_f32", kind="read", sequences=1, tokens=32767, ragged=False, empty=0, kv=12, dim=64,
             kmethod="polarQuant", kbits=4, vmethod="turboQuant", vbits=3, page=48, layout="token", dtype="float32"),
        # one sequence of 777 tokens of a Qwen2.5-1.5B layer: latency
        dict(name="attend_short_bf16", kind="attend", sequences=1, tokens=777, ragged=False, empty=0, kv=2, queries=6, dim=128,
             kmethod="turboQuant", kbits=4, vmethod="turboQuant", vbits=4, page=16, layout="head", softcap=0.0, window=0,
             slopes=False, dtype="bfloat16"),
        # a decode step of 32 ragged sequences of up to 8000 tokens of a Llama-3-8B layer, two of the batch's rows empty
        dict(name="attend_batch_bf16", kind="attend", sequences=32, tokens=8000, ragged=True, empty=2, kv=8, queries=4, dim=128,
             kmethod="turboQuant", kbits=4, vmethod="turboQuant", vbits=4, page=64, layout="head", softcap=0.0, window=0,
             slopes=False, dtype="bfloat16"),
        # the long-context layer: one sequence of 131072 tokens, keys of four bits, values of three
        dict(name="attend_long_bf16", kind="attend", sequences=1, tokens=131072, ragged=False, empty=0, kv=8, queries=4, dim=128,
             kmethod="turboQuant", kbits=4, vmethod="turboQuant", vbits=3, page=64, layout="head", softcap=0.0, window=0,
             slopes=False, dtype="bfloat16"),
        # 64 sequences of heads of 64 with capped scores and a window of 1000 tokens, eight bits, float16
        dict(name="attend_window_f16", kind="attend", sequences=64, tokens=3000, ragged=True, empty=0, kv=4, queries=8, dim=64,
             kmethod="turboQuant", kbits=8, vmethod="turboQuant", vbits=8, page=16, layout="token", softcap=30.0, window=1000,
             slopes=False, dtype="float16"),
        # 200 short sequences with one query head per KV head and a bias by distance, PolarQuant keys
        dict(name="attend_many_bf16", kind="attend", sequences=200, tokens=500, ragged=True, empty=0, kv=12, queries=1, dim=64,
             kmethod="polarQuant", kbits=3, vmethod="turboQuant", vbits=2, page=32, layout="head", softcap=0.0, window=0,
             slopes=True, dtype="bfloat16"),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "append", "read", "attend", "attend", "attend"])
    kmethod, vmethod = (rng.choice(["turboQuant", "turboQuant", "polarQuant"]) for _ in range(2))
    kbits, vbits = (rng.choice([2, 3, 3, 4, 4, 4, 5, 6, 8]) for _ in range(2))
    case = dict(kind=kind, kv=rng.choice([1, 2, 4, 8, 12]), dim=rng.choice([64, 128, 128]), kmethod=kmethod, kbits=kbits,
                vmethod=vmethod, vbits=vbits, page=rng.choice([16, 32, 48, 64, 128]), layout=rng.choice(["head", "head", "token"]))
    if kind == "append":
        tokens = _log(rng, 1, 8192 * 8 // case["kv"] // 4)
        return dict(case, tokens=tokens, padded=rng.randint(0, tokens // 4), queries=rng.randint(1, 8),
                    norm=rng.random() < 0.6, rotary=rng.choice([0, case["dim"], case["dim"], case["dim"] // 2]),
                    dtype=rng.choice(["float32", "float16", "bfloat16", "bfloat16"]))
    sequences = _log(rng, 1, 200)
    most = 1 << (16 if kind == "attend" else 14)
    tokens = _log(rng, 1, max(1, most * 8 // case["kv"] // sequences))
    case.update(sequences=sequences, tokens=min(tokens, most), ragged=rng.random() < 0.7, empty=rng.choice([0, 0, sequences // 8]))
    if kind == "read":
        return dict(case, dtype=rng.choice(["float32", "float16", "bfloat16", "bfloat16"]))
    return dict(case, queries=rng.randint(1, 8), softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                window=rng.choice([0, 0, _log(rng, 1, 4096)]), slopes=rng.random() < 0.3,
                dtype=rng.choice(["float16", "bfloat16", "bfloat16"]))


# ----------------------------------------------------------------------------------------- sizes
def _lengths(case: dict) -> list[int]:
    """Cached tokens of each sequence: spread over 1 .. tokens for a ragged batch, one of them the longest."""
    n, most = case["sequences"], case["tokens"]
    got = [1 + int((most - 1) * ((0.6180339887 * i) % 1.0)) if case["ragged"] and i else most for i in range(n)]
    return [0 if i >= n - case["empty"] else t for i, t in enumerate(got)]


def _seen(case: dict) -> int:
    """Tokens that the new tokens attend to."""
    return sum(min(t, case["window"] or t) for t in _lengths(case))


def _stride(dim: int, bits: int) -> int:
    return dim * bits // 8


def work(case: dict) -> dict:
    kv, d, elem = case["kv"], case["dim"], DTYPES[case["dtype"]].itemsize
    cached = kv * (_stride(d, case["kbits"]) + _stride(d, case["vbits"]) + 8)   # one token's codes and scales
    if case["kind"] == "append":
        n, heads = case["tokens"] - case["padded"], kv * case["queries"]
        rows = (2 * heads + 2 * kv) * n + 2 * heads * case["padded"]
        tables = 8 * case["rotary"] * case["tokens"] + 16 * case["tokens"]
        return {"bytes": rows * d * elem + cached * n + tables,
                "flops": n * 2 * kv * d * (math.log2(d) + 4) + (heads + kv) * n * d * 6}
    if case["kind"] == "read":
        n = sum(_lengths(case))
        return {"bytes": n * (cached + 2 * kv * d * elem) + 4 * n // case["page"], "flops": n * 2 * kv * d * (math.log2(d) + 2)}
    n, heads = _seen(case), kv * case["queries"]
    return {"bytes": n * cached + 2 * case["sequences"] * heads * d * elem + 4 * n // case["page"], "flops": 4.0 * n * heads * d}


# ----------------------------------------------------------------------------------------- the codes
_books: dict | None = None


def _book(dim: int, bits: int):
    global _books
    if _books is None:
        _books = json.loads((Path(__file__).resolve().parent.parent / "pitch_amd" / "data" / "codebooks.json").read_text())
    return torch.tensor(_books[f"{dim}_{bits}"], dtype=torch.float32, device=DEVICE)


def _signs(dim: int):
    """The rotation's random signs: the last bit of a 32-bit hash of seed + coordinate."""
    m = 0xFFFFFFFF
    state = ((torch.arange(dim) + SEED) & m) * 747796405 + 2891336453 & m
    word = ((state >> ((state >> 28) + 4)) ^ state) * 277803737 & m
    return torch.where(((word >> 22) ^ word) & 1 == 1, 1.0, -1.0).to(DEVICE)


def _hadamard(dim: int, dtype):
    i = torch.arange(dim)
    x = i[:, None] & i[None, :]
    x = x ^ (x >> 4)
    x = x ^ (x >> 2)
    x = x ^ (x >> 1)
    return torch.where(x & 1 == 1, -1.0, 1.0).to(DEVICE, dtype)


def _packed(codes, bits: int):
    """Codes [..., dim] as bytes [..., dim * bits / 8]: code i at bits [i bits, (i + 1) bits) of a little-endian stream."""
    b = (codes[..., None] >> torch.arange(bits, device=DEVICE)) & 1
    b = b.reshape(*codes.shape[:-1], -1, 8)
    return (b << torch.arange(8, device=DEVICE)).sum(-1).to(torch.uint8)


def _unpacked(stream, dim: int, bits: int):
    """The codes [..., dim] of bytes [..., dim * bits / 8]."""
    b = (stream[..., None] >> torch.arange(8, device=DEVICE, dtype=torch.uint8)) & 1
    b = b.reshape(*stream.shape[:-1], dim, bits)
    return (b << torch.arange(bits, device=DEVICE, dtype=torch.uint8)).sum(-1, dtype=torch.int32)


def _quantised(x, method: str, bits: int):
    """(codes, scales) of vectors [..., dim], in the vectors' own float type."""
    dim = x.shape[-1]
    y = (x * _signs(dim)) @ _hadamard(dim, x.dtype) / math.sqrt(dim)
    if method == "turboQuant":
        norm = x.square().sum(-1).sqrt()
        book = _book(dim, bits)
        edges = (0.5 * (book[1:] + book[:-1])).to(x.dtype)
        u = y / torch.where(norm > 0, norm, 1.0)[..., None]
        return torch.searchsorted(edges, u), norm
    a, c = y[..., 0::2], y[..., 1::2]
    levels = 1 << bits
    r = torch.hypot(a, c)
    top = r.amax(-1)
    rq = (r / torch.where(top > 0, top, 1.0)[..., None] * (levels - 1) + 0.5).floor().clamp(0, levels - 1)
    turn = torch.remainder(torch.atan2(c, a), 2 * math.pi) / (2 * math.pi)
    tq = torch.remainder((turn * levels + 0.5).floor(), levels)
    return torch.stack([rq, tq], -1).flatten(-2).to(torch.int64), top


def _decoded(stream, scales, dim: int, method: str, bits: int):
    """The float32 vectors that codes and scales stand for."""
    codes = _unpacked(stream, dim, bits)
    if method == "turboQuant":
        y = _book(dim, bits)[codes]
    else:
        r = codes[..., 0::2].float() / ((1 << bits) - 1)
        t = codes[..., 1::2].double() * (2 * math.pi / (1 << bits))
        y = torch.stack([r * torch.cos(t).float(), r * torch.sin(t).float()], -1).flatten(-2)
    y = y @ _hadamard(dim, torch.float32)
    return y * (_signs(dim) / math.sqrt(dim)) * scales[..., None]


# ----------------------------------------------------------------------------------------- inputs
def _keys(gen, *shape):
    """Keys as a projection gives them: uneven channels, a few of them large, an offset per head."""
    dim = shape[-1]
    x = torch.randn(shape, generator=gen, device=DEVICE)
    s = torch.exp(0.4 * torch.randn((shape[-2], dim), generator=gen, device=DEVICE))
    s[:, :: max(1, dim // 4)] *= 4.0
    return (x + 0.5 * torch.randn((shape[-2], dim), generator=gen, device=DEVICE)) * s


def _values(gen, *shape):
    """Heavy-tailed values, each head with a scale of its own."""
    z = torch.randn(shape, generator=gen, device=DEVICE)
    tail = torch.randn(shape[:-1] + (5,), generator=gen, device=DEVICE).square().mean(-1, keepdim=True).clamp(min=0.05)
    return z / tail.sqrt() * torch.exp(torch.randn((shape[-2], 1), generator=gen, device=DEVICE) * 0.5)


def _pool(case: dict, pages: int, bits: int, gen):
    """An allocated pool with what earlier sequences left in it: (codes, scales)."""
    lead = (pages, case["kv"], case["page"]) if case["layout"] == "head" else (pages, case["page"], case["kv"])
    codes = torch.randint(0, 256, lead + (_stride(case["dim"], bits),), generator=gen, device=DEVICE, dtype=torch.uint8)
    return codes, torch.rand(lead, generator=gen, device=DEVICE) * 10 + 0.1


def _by_head(case: dict, t):
    """The pool as [page][slot][head]."""
    return t if case["layout"] == "token" else t.transpose(1, 2)


def _rotary(positions: int, dim: int):
    inv = 1.0 / 1e6 ** (torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)
    angle = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * inv
    return tuple(torch.cat([f(angle)] * 2, 1).float().contiguous() for f in (torch.cos, torch.sin))


def _cache(case: dict, s: dict):
    import pitch_amd as P
    q = P.PITCH(SEED)
    kc = q.config(case["kmethod"], case["dim"], case["kbits"])
    vc = q.config(case["vmethod"], case["dim"], case["vbits"])
    return P.PagedCache(q, kc, vc, pages=s["pages"], pageSize=case["page"], kvHeads=case["kv"], layout=case["layout"],
                        keyCodes=s["key_codes"], keyScales=s["key_scales"], valueCodes=s["value_codes"],
                        valueScales=s["value_scales"])


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kv, d, page, dtype = case["kv"], case["dim"], case["page"], DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "append":
        n, heads = case["tokens"], kv * case["queries"]
        s["pages"] = -(-n // page) + 3
        for name, bits in (("key", case["kbits"]), ("value", case["vbits"])):
            s[name + "_codes"], s[name + "_scales"] = _pool(case, s["pages"], bits, gen)
        # queries, keys and values are slices of the projection's output
        qkv = torch.empty((n, heads + 2 * kv, d), device=DEVICE, dtype=dtype)
        qkv[:, :heads] = torch.randn((n, heads, d), generator=gen, device=DEVICE).to(dtype)
        qkv[:, heads:heads + kv] = _keys(gen, n, kv, d).to(dtype)
        qkv[:, heads + kv:] = _values(gen, n, kv, d).to(dtype)
        s["queries"], s["keys"], s["values"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        s["out"] = torch.zeros((n, heads, d), device=DEVICE, dtype=dtype)
        slots = torch.randperm(s["pages"] * page, generator=gen, device=DEVICE)[:n]
        if case["padded"]:
            slots[n - case["padded"]:] = -1
        s["slots"] = slots
        s["norms"] = [(1 + 0.2 * torch.randn(d, generator=gen, device=DEVICE)).to(dtype) if case["norm"] else None for _ in range(2)]
        s["cos"], s["sin"], s["positions"] = None, None, None
        if case["rotary"]:
            s["cos"], s["sin"] = _rotary(max(n, 2048), case["rotary"])
            s["positions"] = torch.randint(0, s["cos"].shape[0], (n,), generator=gen, device=DEVICE)
        if own:
            import pitch_amd as P
            s["call"] = P.PagedAppend(_cache(case, s), s["keys"], s["values"], s["slots"], queries=s["queries"],
                                      queriesOut=s["out"], queryNorm=s["norms"][0], keyNorm=s["norms"][1], eps=EPS,
                                      cos=s["cos"], sin=s["sin"], positions=s["positions"])
        return s
    lengths = _lengths(case)
    used = [-(-t // page) for t in lengths]
    s["pages"] = sum(used) + 3
    # a pool whose pages hold what keys and values quantise to, handed out to the sequences in no order
    for name, method, bits, make in (("key", case["kmethod"], case["kbits"], _keys), ("value", case["vmethod"], case["vbits"], _values)):
        x = make(gen, s["pages"] * page, kv, d)
        codes, scales = _quantised(x, method, bits)
        del x
        codes, scales = _packed(codes.to(torch.uint8), bits).view(s["pages"], page, kv, -1), scales.view(s["pages"], page, kv)
        s[name + "_codes"], s[name + "_scales"] = (t if case["layout"] == "token" else t.transpose(1, 2).contiguous()
                                                   for t in (codes, scales))
    ids = torch.randperm(s["pages"], generator=gen, device=DEVICE).to(torch.int32)
    at, width = np.concatenate([[0], np.cumsum(used)]), max(max(used), 1)
    col = torch.arange(width, device=DEVICE)
    first = torch.tensor(at[:-1], device=DEVICE)
    s["tables"] = torch.where(col < torch.tensor(used, device=DEVICE)[:, None], ids[(first[:, None] + col).clamp(max=s["pages"] - 1)],
                              -1).to(torch.int32)
    s["lengths"] = torch.tensor(lengths, device=DEVICE, dtype=torch.int32)
    if case["kind"] == "read":
        rows = sum(lengths)
        s["starts"] = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), device=DEVICE, dtype=torch.int32)
        s["rows"] = rows
        s["keys"], s["values"] = (torch.zeros((rows, kv, d), device=DEVICE, dtype=dtype) for _ in range(2))
        if own:
            import pitch_amd as P
            s["call"] = P.PagedDecode(_cache(case, s), s["tables"], s["starts"], keysOut=s["keys"], valuesOut=s["values"])
        return s
    heads = kv * case["queries"]
    s["queries"] = (torch.randn((case["sequences"], heads, d), generator=gen, device=DEVICE) * 1.2).to(dtype)
    s["out"] = torch.zeros((case["sequences"], heads, d), device=DEVICE, dtype=dtype)
    s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, heads + 1, device=DEVICE) / heads)).float() if case["slopes"] else None
    if own:
        import pitch_amd as P
        s["call"] = P.PagedAttention(_cache(case, s), s["queries"], s["tables"], s["lengths"], s["out"], scale=1 / math.sqrt(d),
                                     softcap=case["softcap"], window=case["window"], slopes=s["slopes"])
    return s


# ----------------------------------------------------------------------------------------- the operators
def _normed(x, weight):
    """x times the weights, and the factor 1 / rms that belongs to it (kept apart: it does not change a code)."""
    if weight is None:
        return x, torch.ones_like(x[..., 0])
    return x * weight, (x.square().mean(-1) + EPS).rsqrt()


def _rotated(x, s):
    """x with its first `rotary` coordinates turned to the tokens' positions."""
    if s["cos"] is None:
        return x
    n = s["cos"].shape[1]
    cos, sin = (s[t][s["positions"]][:, None].to(x.dtype) for t in ("cos", "sin"))
    head = x[..., :n]
    half = torch.cat([-head[..., n // 2:], head[..., : n // 2]], -1)
    return torch.cat([head * cos + half * sin, x[..., n:]], -1)


def _append(s: dict):
    case = s["case"]
    q, r = _normed(s["queries"].float(), None if s["norms"][0] is None else s["norms"][0].float())
    s["out"].copy_(_rotated(q, s) * r[..., None])
    # in 64 bits: a value next to an edge of two codes has to fall on the right side
    k, r = _normed(s["keys"].double(), None if s["norms"][1] is None else s["norms"][1].double())
    codes = {"key": _quantised(_rotated(k, s), case["kmethod"], case["kbits"]),
             "value": _quantised(s["values"].double(), case["vmethod"], case["vbits"])}
    n = case["tokens"] - case["padded"]
    page, slot = s["slots"][:n] // case["page"], s["slots"][:n] % case["page"]
    _by_head(case, s["key_codes"])[page, slot] = _packed(codes["key"][0], case["kbits"])[:n]
    _by_head(case, s["key_scales"])[page, slot] = (codes["key"][1] * r)[:n].float()
    _by_head(case, s["value_codes"])[page, slot] = _packed(codes["value"][0], case["vbits"])[:n]
    _by_head(case, s["value_scales"])[page, slot] = codes["value"][1][:n].float()


def _tokens(s: dict, name: str, page, slot):
    case = s["case"]
    bits, method = (case["kbits"], case["kmethod"]) if name == "key" else (case["vbits"], case["vmethod"])
    return _decoded(_by_head(case, s[name + "_codes"])[page, slot], _by_head(case, s[name + "_scales"])[page, slot], case["dim"],
                    method, bits)


def _read(s: dict):
    row = torch.arange(s["rows"], device=DEVICE)
    seq = torch.searchsorted(s["starts"], row, right=True) - 1
    token = row - s["starts"][seq]
    page, slot = s["tables"][seq, token // s["case"]["page"]].long(), token % s["case"]["page"]
    s["keys"].copy_(_tokens(s, "key", page, slot))
    s["values"].copy_(_tokens(s, "value", page, slot))


def _attend(s: dict):
    case = s["case"]
    length = s["lengths"].long()[:, None]
    token = torch.arange(case["tokens"], device=DEVICE)[None]
    last = length - 1
    if case["window"]:       # only the window's tokens are looked at
        token = (length - case["window"]).clamp(min=0) + token[:, : min(case["window"], case["tokens"])]
    seen = token < length
    token = torch.where(seen, token, 0)
    page, slot = torch.gather(s["tables"], 1, token // case["page"]).clamp(min=0).long(), token % case["page"]
    k, v = (_tokens(s, name, page, slot).transpose(1, 2) for name in ("key", "value"))     # [sequence][head][token][dim]
    q = s["queries"].float().view(case["sequences"], case["kv"], case["queries"], case["dim"])
    score = q @ k.transpose(2, 3).contiguous() / math.sqrt(case["dim"])
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    if s["slopes"] is not None:
        score = score + s["slopes"].view(1, case["kv"], case["queries"], 1) * (token - last)[:, None, None, :]
    score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = p @ v.contiguous() / torch.where(total > 0, total, 1.0)
    s["out"].copy_(o.view(s["out"].shape))


def run(s: dict):
    kind = s["case"]["kind"]
    if own:
        s["call"].enqueue()
    elif kind == "append":
        _append(s)
    elif kind == "read":
        _read(s)
    else:
        _attend(s)
    if kind == "append":
        return {"queries": s["out"], "key_codes": s["key_codes"], "key_scales": s["key_scales"], "value_codes": s["value_codes"],
                "value_scales": s["value_scales"]}
    return {"keys": s["keys"], "values": s["values"]} if kind == "read" else s["out"]


# ----------------------------------------------------------------------------------------- the definition, in 64 bits
def _sylvester(dim: int):
    h = torch.ones((1, 1), dtype=torch.float64, device=DEVICE)
    while h.shape[0] < dim:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    sign = []
    for i in range(dim):
        st = ((SEED + i) % 2 ** 32 * 747796405 + 2891336453) % 2 ** 32
        w = ((st >> ((st >> 28) + 4)) ^ st) * 277803737 % 2 ** 32
        sign.append(1.0 if ((w >> 22) ^ w) % 2 else -1.0)
    return h * torch.tensor(sign, dtype=torch.float64, device=DEVICE) / math.sqrt(dim)   # codes' domain -> vectors


def _vectors64(stream, scale, dim: int, method: str, bits: int):
    """What rows of packed codes [n, stride] and scales [n] stand for, bit by bit of the stream's 32-bit words."""
    w = stream.contiguous().view(torch.int32).to(torch.int64) & 0xFFFFFFFF
    y = torch.empty((w.shape[0], dim), dtype=torch.float64, device=DEVICE)
    book = _book(dim, bits).double()
    for i in range(dim):
        lo, sh = i * bits // 32, i * bits % 32
        code = w[:, lo] >> sh
        if sh + bits > 32:
            code = code | (w[:, lo + 1] << (32 - sh))
        code = code & ((1 << bits) - 1)
        if method == "turboQuant":
            y[:, i] = book[code]
        elif i % 2 == 0:
            y[:, i] = code.double() / ((1 << bits) - 1)
        else:
            angle = code.double() * 2 * math.pi / (1 << bits)
            y[:, i] = y[:, i - 1] * torch.sin(angle)
            y[:, i - 1] *= torch.cos(angle)
    return (y @ _sylvester(dim)) * scale.double()[:, None]


def _sequence64(s: dict, b: int, tokens: int, name: str, first: int = 0):
    """Tokens [first, first + tokens) of sequence b: [token][head][dim]."""
    case = s["case"]
    bits, method = (case["kbits"], case["kmethod"]) if name == "key" else (case["vbits"], case["vmethod"])
    t = torch.arange(first, first + tokens, device=DEVICE)
    page, slot = s["tables"][b].long()[t // case["page"]], t % case["page"]
    c, n = (_by_head(case, s[name + x])[page, slot] for x in ("_codes", "_scales"))
    return _vectors64(c.reshape(tokens * case["kv"], -1), n.reshape(-1), case["dim"], method, bits).view(tokens, case["kv"], -1)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kv, d = case["kv"], case["dim"]
    if case["kind"] == "append":
        def turned(x, weight):
            x = x.double()
            y = x if weight is None else x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS) * weight.double()
            n = case["rotary"]
            if not n:
                return y
            z = y.clone()
            for i in range(n // 2):
                j = i + n // 2
                c, w = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]
                z[..., i] = y[..., i] * c[:, None, i] - y[..., j] * w[:, None, i]
                z[..., j] = y[..., j] * c[:, None, j] + y[..., i] * w[:, None, j]
            return z

        n, scales = case["tokens"] - case["padded"], {}
        for name, x, method in (("key", turned(s["keys"], s["norms"][1]), case["kmethod"]), ("value", s["values"].double(), case["vmethod"])):
            if method == "turboQuant":
                size = torch.linalg.vector_norm(x, dim=-1)
            else:
                y = x @ _sylvester(d).T
                size = torch.sqrt(y[..., 0::2] ** 2 + y[..., 1::2] ** 2).amax(-1)
            pool = s[name + "_scales"].double()
            at = _by_head(case, pool)
            at[s["slots"][:n] // case["page"], s["slots"][:n] % case["page"]] = size[:n]
            scales[name] = pool
        return {"queries": turned(s["queries"], s["norms"][0]), "key_codes": None, "key_scales": scales["key"], "value_codes": None,
                "value_scales": scales["value"]}
    lengths = _lengths(case)
    if case["kind"] == "read":
        return {name + "s": torch.cat([_sequence64(s, b, t, name) for b, t in enumerate(lengths) if t]) for name in ("key", "value")}
    out = torch.zeros((case["sequences"], kv, case["queries"], d), dtype=torch.float64, device=DEVICE)
    for b, t in enumerate(lengths):
        if not t:
            continue
        first = max(0, t - case["window"]) if case["window"] else 0
        k, v = (_sequence64(s, b, t - first, name, first) for name in ("key", "value"))
        for h in range(kv):
            z = s["queries"][b, h * case["queries"]:(h + 1) * case["queries"]].double() @ k[:, h].T.contiguous() / math.sqrt(d)
            if case["softcap"]:
                z = torch.tanh(z / case["softcap"]) * case["softcap"]
            if s["slopes"] is not None:
                z = z - s["slopes"][h * case["queries"]:(h + 1) * case["queries"], None].double() * torch.arange(t - 1 - first, -1, -1, device=DEVICE)
            out[b, h] = torch.softmax(z, -1) @ v[:, h].contiguous()
    return out.view(case["sequences"], kv * case["queries"], d)
