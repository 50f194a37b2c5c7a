"""The paged cache's operators against float64 on the CPU: PagedAppend (norms, rotation, quantisation into slots), PagedDecode
(reading ranges back through page tables) and PagedAttention (one new token of every sequence over its pages).

Bars. Codes are computed in float64, so they equal the oracle's except where a value lies within the oracle's near-boundary
band. A scale is a float64 value rounded once to float32: 2^-24. Queries pass through float32: their last rounding (half a
step of their type) plus 16 float32 roundings of the products' magnitudes (the sum of squares of 64 or 128 in at most 12
levels, its root, the division, three products and a sum). Read-back vectors are the bytes of enqueueDecode. Attention: the
output's last rounding, plus what rounding one table value to float16 (2^-11) can do: delta = 2^-11 scale |q| |k| moves a
score, exp(2 delta) - 1 a weight relative to the others, and 2^-11 a value, all relative to sum p |v|; float32 sums of up to
2^17 terms and the exponentials add less than 2^-14 to that. All in the 2-norm per query head.
"""
import math

import numpy as np
import pytest

from oracle import pitch_oracle as O

pytestmark = pytest.mark.gpu

HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
# Below 2^-14 a float16 is subnormal: its step stays 2^-24 and half of it, 2^-25, is more than 2^-11 of the value.
SMALLEST_HALF_STEP = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}


def _rounding(dtype, x):
    """How far rounding x to the type may be off."""
    return np.maximum(HALF_STEP[dtype] * np.abs(x), SMALLEST_HALF_STEP[dtype])


def _torch_dtype(name):
    import torch
    return getattr(torch, name)


def _cache(q, kcfg, vcfg, pages, page, heads, layout, fill=0xA5):
    import torch
    import pitch_amd as P
    c = P.PagedCache(q, kcfg, vcfg, pages=pages, pageSize=page, kvHeads=heads, layout=layout)
    for t in (c.keyCodes, c.valueCodes):
        t.fill_(fill)
    for t in (c.keyScales, c.valueScales):
        t.fill_(-7.0)
    torch.cuda.synchronize()
    return c


def _by_slot(cache, t):
    """A pool's buffer as [slot of the pool][head]... on the CPU."""
    t = t if cache.layout == "token" else t.transpose(1, 2)
    return t.reshape((cache.pages * cache.pageSize, cache.kvHeads) + tuple(t.shape[3:])).cpu().numpy()


def _near(method, X, b, seed):
    return O.turbo_near_boundary(O.turbo_rotated(X, seed), b) if method == "turboQuant" else O.polar_near_boundary(X, b, seed)


def _check_pool(cfg, codes, scales, X):
    """codes [n][stride], scales [n] against the oracle's encoding of X [n][dim] (float64)."""
    ref, size = O.ENCODERS[cfg.method.value](X, cfg.bits, cfg.seed)
    got = O.unpack_codes(codes.tobytes(), X.shape[0], cfg.dim, cfg.bits)
    bad = (got != ref) & ~_near(cfg.method.value, X, cfg.bits, cfg.seed)
    assert not bad.any(), f"{int(bad.sum())} codes differ away from any edge"
    assert np.abs(scales - size).max(initial=0) <= 2.0 ** -24 * 1.001 * max(size.max(initial=0), 1e-30)


def _rotate(x, cos, sin, pos):
    """(rotated, sum of the products' magnitudes) of x [tokens][heads][dim]; tables float32 [positions][n]."""
    n = cos.shape[1]
    c, s = cos[pos].astype(np.float64)[:, None], sin[pos].astype(np.float64)[:, None]
    h = x[..., :n]
    half = np.concatenate([-h[..., n // 2:], h[..., :n // 2]], -1)
    out, mag = x.copy(), np.abs(x)
    out[..., :n] = h * c + half * s
    mag[..., :n] = np.abs(h * c) + np.abs(half * s)
    return out, mag


def _normed(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


APPENDS = [
    # dim, kv, q heads, tokens, (method, bits) of keys and values, page, layout, dtype, norm, rotary
    (128, 8, 32, 1, ("turboQuant", 4), ("turboQuant", 4), 16, "head", "bfloat16", True, 128),
    (128, 2, 12, 37, ("turboQuant", 4), ("turboQuant", 3), 64, "head", "bfloat16", True, 128),
    (128, 3, 3, 130, ("turboQuant", 2), ("turboQuant", 8), 48, "token", "float16", True, 64),
    (128, 1, 0, 5, ("turboQuant", 5), ("polarQuant", 5), 32, "token", "float32", False, 0),
    (128, 8, 8, 257, ("polarQuant", 4), ("polarQuant", 3), 16, "head", "float32", True, 128),
    (128, 2, 2, 33, ("polarQuant", 8), ("turboQuant", 6), 80, "head", "float16", False, 32),
    (64, 12, 12, 65, ("turboQuant", 3), ("turboQuant", 7), 32, "head", "float32", True, 64),
    (64, 4, 28, 19, ("polarQuant", 6), ("polarQuant", 7), 16, "token", "bfloat16", False, 16),
    (64, 1, 1, 3, ("polarQuant", 2), ("turboQuant", 2), 16, "head", "bfloat16", False, 0),
    (64, 5, 10, 3000, ("turboQuant", 4), ("turboQuant", 5), 128, "token", "bfloat16", True, 32),
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"d{c[0]}-kv{c[1]}-q{c[2]}-n{c[3]}-{c[4][0][0]}{c[4][1]}{c[5][0][0]}{c[5][1]}-{c[8]}")
def test_append(q, case):
    import torch
    import pitch_amd as P
    d, kv, nq, n, (km, kb), (vm, vb), page, layout, dtype, norm, rotary = case
    dt, dev = _torch_dtype(dtype), q.device
    kcfg, vcfg = P.QuantConfig(km, d, kb, 5), P.QuantConfig(vm, d, vb, 6)
    pages = -(-n // page) + 2
    cache = _cache(q, kcfg, vcfg, pages, page, kv, layout)
    g = torch.Generator().manual_seed(n * d + kb)
    # keys, values and queries as slices of one projection
    qkv = (torch.randn(n, nq + 2 * kv + 1, d, generator=g) * torch.exp(torch.randn(d, generator=g) * 0.5)).to(dt)
    on = qkv.to(dev)
    keys, values = on[:, nq:nq + kv], on[:, nq + kv:nq + 2 * kv]
    slots = torch.randperm(pages * page, generator=g)[:n]
    skipped = [i for i in range(n) if i % 7 == 3]
    slots[skipped] = torch.tensor([-1 - (i % 2) * 2 ** 40 if i % 3 else pages * page + i for i in skipped], dtype=torch.int64)
    more, w = {}, [torch.ones(d)] * 2
    if nq:
        out = torch.full((n, nq, d), -3.0, dtype=dt, device=dev)
        more.update(queries=on[:, :nq], queriesOut=out)
    if norm:
        w = [(1 + 0.3 * torch.randn(d, generator=g)).to(dt) for _ in range(2)]
        more.update(keyNorm=w[1].to(dev), eps=1e-5)
        if nq:
            more.update(queryNorm=w[0].to(dev))
    lost = []
    if rotary:
        angle = torch.arange(50, dtype=torch.float64)[:, None] * torch.exp(-torch.arange(rotary // 2) * 0.2)
        cos, sin = (torch.cat([f(angle)] * 2, 1).float() for f in (torch.cos, torch.sin))
        sin[:, rotary // 2:] *= 1.25     # the two halves of the tables are read each for itself
        pos = torch.randint(0, 50, (n,), generator=g)
        lost = [i for i in range(n) if i % 11 == 5]
        pos[lost] = torch.tensor([50 if i % 2 else -1 for i in lost], dtype=torch.int64)
        more.update(cos=cos.to(dev), sin=sin.to(dev), positions=pos.to(dev))
    cache.enqueueAppend(keys, values, slots.to(dev), **more)
    torch.cuda.synchronize()

    x = qkv.double().numpy()
    xq, xk, xv = x[:, :nq], x[:, nq:nq + kv], x[:, nq + kv:nq + 2 * kv]
    if norm:
        xk = _normed(xk, w[1].double().numpy(), float(np.float32(1e-5)))
        xq = _normed(xq, w[0].double().numpy(), float(np.float32(1e-5)))
    mag = np.abs(xq)
    if rotary:
        safe = pos.clamp(0, 49).numpy()
        xk, _ = _rotate(xk, cos.numpy(), sin.numpy(), safe)
        xq, mag = _rotate(xq, cos.numpy(), sin.numpy(), safe)
    kept = [i for i in range(n) if i not in set(skipped) | set(lost)]
    at = slots[kept].numpy()
    for cfg, codes, scales, X in ((kcfg, cache.keyCodes, cache.keyScales, xk), (vcfg, cache.valueCodes, cache.valueScales, xv)):
        codes, scales = _by_slot(cache, codes), _by_slot(cache, scales)
        if kept:
            _check_pool(cfg, codes[at].reshape(-1, cfg.codeStride), scales[at].reshape(-1).astype(np.float64),
                        X[kept].reshape(-1, d))
        rest = np.setdiff1d(np.arange(pages * page), at)
        assert (codes[rest] == 0xA5).all() and (scales[rest] == -7.0).all(), "a slot that was not written has changed"
    if nq:
        got = out.double().cpu().numpy()
        there = [i for i in range(n) if i not in set(lost)]
        bar = _rounding(dtype, xq) + 16 * 2.0 ** -24 * mag
        assert (np.abs(got - xq)[there] <= bar[there] * 1.001 + 1e-30).all()
        assert (got[lost] == -3.0).all()


@pytest.mark.parametrize("method,bits,d,dtype", [("turboQuant", 4, 128, "bfloat16"), ("turboQuant", 3, 64, "float32"),
                                                 ("polarQuant", 4, 128, "float16"), ("polarQuant", 8, 64, "bfloat16"),
                                                 ("turboQuant", 8, 128, "float32")])
def test_append_and_read_are_the_contiguous_codec(q, method, bits, d, dtype):
    """Without norm and rotation a page holds what enqueueEncode writes, and reads back as the bytes of enqueueDecode."""
    import torch
    import pitch_amd as P
    dev, dt, n, kv, page = q.device, _torch_dtype(dtype), 203, 3, 32
    cfg = P.QuantConfig(method, d, bits, 99)
    cache = _cache(q, cfg, cfg, 9, page, kv, "head")
    x = torch.randn(n, kv, d, device=dev, generator=torch.Generator(device=dev).manual_seed(d)).to(dt)
    x[5] = 0.0      # a zero vector
    slots = torch.randperm(9 * page, device=dev)[:n]
    cache.enqueueAppend(x, x, slots)
    codes = torch.empty(n * kv * cfg.codeStride, dtype=torch.uint8, device=dev)
    scales = torch.empty(n * kv, dtype=torch.float32, device=dev)
    q.enqueueEncode(x, codes, scales, n * kv, cfg)
    at = slots.cpu().numpy()
    assert np.array_equal(_by_slot(cache, cache.keyCodes)[at].reshape(-1), codes.cpu().numpy())
    assert np.array_equal(_by_slot(cache, cache.valueCodes)[at].reshape(-1), codes.cpu().numpy())
    assert np.allclose(_by_slot(cache, cache.keyScales)[at].reshape(-1), scales.cpu().numpy(), rtol=2.0 ** -22, atol=0)
    # the pool's tokens in slot order through a table of all pages
    pool = torch.zeros(9 * page, kv, d, device=dev, dtype=dt)
    full = torch.zeros(9 * page * kv, dtype=torch.float32, device=dev)
    cache.keyScales.clamp_(min=0.0)
    cache.enqueueDecode(torch.arange(9, dtype=torch.int32, device=dev)[None], torch.tensor([0, 9 * page], dtype=torch.int32, device=dev),
                        keysOut=pool)
    ref = torch.empty(9 * page * kv, d, device=dev, dtype=dt)
    flat = torch.from_numpy(np.ascontiguousarray(_by_slot(cache, cache.keyCodes)).reshape(-1)).to(dev)
    full.copy_(torch.from_numpy(np.ascontiguousarray(_by_slot(cache, cache.keyScales)).reshape(-1)))
    q.enqueueDecode(flat, full, ref, 9 * page * kv, cfg)
    torch.cuda.synchronize()
    assert torch.equal(pool.view(-1, d), ref)


READS = [
    # dim, kv, (method, bits), page, layout, dtype, lengths, first tokens?
    (128, 8, ("turboQuant", 4), 16, "head", "bfloat16", [1], False),
    (128, 2, ("turboQuant", 3), 64, "token", "float32", [0, 5, 0, 64, 65, 0], False),
    (64, 3, ("polarQuant", 3), 48, "head", "float16", [17, 100, 3, 250], True),
    (64, 1, ("turboQuant", 7), 32, "token", "bfloat16", [1000, 1, 31], True),
    (128, 1, ("polarQuant", 5), 16, "head", "float32", list(range(40)), True),
    (128, 4, ("turboQuant", 2), 32, "head", "bfloat16", [3] * 1300, False),
]


@pytest.mark.parametrize("case", READS, ids=lambda c: f"d{c[0]}-kv{c[1]}-{c[2][0][0]}{c[2][1]}-p{c[3]}-{c[5]}-{len(c[6])}seq")
def test_read(q, case):
    import torch
    import pitch_amd as P
    d, kv, (method, bits), page, layout, dtype, lengths, offset = case
    dev, dt = q.device, _torch_dtype(dtype)
    rng = np.random.default_rng(d + bits + len(lengths))
    first = [int(rng.integers(0, 70)) if offset else 0 for _ in lengths]
    width = max(-(-(f + n) // page) for f, n in zip(first, lengths)) + 1
    pages = len(lengths) * width + 2
    kcfg = P.QuantConfig(method, d, bits, 7)
    vcfg = P.QuantConfig("turboQuant", d, 4, 8)
    cache = _cache(q, kcfg, vcfg, pages, page, kv, layout)
    codes = {}
    for name, cfg in (("key", kcfg), ("value", vcfg)):
        t = getattr(cache, name + "Codes")
        t.copy_(torch.from_numpy(rng.integers(0, 256, tuple(t.shape), dtype=np.uint8)))
        getattr(cache, name + "Scales").copy_(torch.from_numpy(np.exp(rng.normal(size=tuple(t.shape[:3]))).astype(np.float32)))
        c, s = _by_slot(cache, t), _by_slot(cache, getattr(cache, name + "Scales"))
        codes[name] = (c, s, cfg)
    tables = rng.permutation(pages)[:len(lengths) * width].reshape(len(lengths), width).astype(np.int32)
    starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32) + 2     # two rows in front, some behind
    rows = int(starts[-1]) + 9
    bad = None
    if len(lengths) > 2:      # a page outside the pool: its rows stay
        bad = (1, (first[1] + lengths[1] // 2) // page)
        tables[bad] = -1 if offset else pages
    wide = torch.full((rows, kv + 1, d), -5.0, dtype=dt, device=dev)
    keys = wide[:, :kv]                                                          # strided
    values = torch.full((kv, rows, d), -5.0, dtype=dt, device=dev).transpose(0, 1)  # head-major
    more = {"firstTokens": torch.tensor(first, dtype=torch.int32, device=dev)} if offset else {}
    cache.enqueueDecode(torch.from_numpy(tables).to(dev), torch.from_numpy(starts).to(dev), keysOut=keys, valuesOut=values, **more)
    torch.cuda.synchronize()
    expect, written = np.full((rows,), -1, np.int64), np.zeros(rows, bool)
    for b, n in enumerate(lengths):
        for i in range(n):
            t = first[b] + i
            if (b, t // page) != bad:
                expect[starts[b] + i] = tables[b, t // page] * page + t % page
    written = expect >= 0
    for name, got in (("key", keys), ("value", values)):
        c, s, cfg = codes[name]
        got = got.double().cpu().numpy()
        assert (got[~written] == -5.0).all()
        if written.any():
            at = expect[written]
            u = O.unpack_codes(c[at].tobytes(), len(at) * kv, d, cfg.bits)
            ref = O.DECODERS[cfg.method.value](u, s[at].reshape(-1).astype(np.float64), cfg.bits, cfg.seed).reshape(-1, kv, d)
            # d float32 butterflies: log2(d) + 3 roundings of the vector's norm; then the type's own
            size = np.linalg.norm(ref, axis=-1, keepdims=True)
            assert (np.abs(got[written] - ref) <= _rounding(dtype, ref) + 10 * 2.0 ** -24 * size).all()
    assert (wide[:, kv] == -5.0).all()


@pytest.mark.parametrize("d,kv,nq,method,dtype,layout", [(128, 5, 7, "turboQuant", "bfloat16", "head"),
                                                         (64, 6, 9, "turboQuant", "float32", "token"),
                                                         (128, 7, 2, "polarQuant", "float16", "token"),
                                                         (64, 9, 0, "turboQuant", "float16", "head")])
def test_long_calls_equal_short_ones(q, d, kv, nq, method, dtype, layout):
    """Long calls give a workgroup four heads of its tokens, here with groups that are not full, short calls one: the same codes,
    scales, queries and vectors, bit for bit, and rows and slots that are not named stay as they were."""
    import torch
    n, page, dt = 12000, 64, _torch_dtype(dtype)
    kcfg, vcfg = q.config(method, d, 5), q.config("turboQuant", d, 4)
    torch.manual_seed(d + kv)
    x = torch.randn(n, kv + nq, d, device="cuda").to(dt)
    keys, values, queries = x[:, :kv], x[:, :kv].flip(0).contiguous(), x[:, kv:]
    cos, sin = (torch.rand(n, d // 2, device="cuda") for _ in range(2))
    weight = (torch.rand(d, device="cuda") + 0.5).to(dt)
    pages = n // page + 2
    slots = torch.randperm(pages * page, device="cuda")[:n]
    slots[5::11] = -1
    results = []
    for step in (n, 500):
        cache = _cache(q, kcfg, vcfg, pages, page, kv, layout)
        out = torch.full((n, max(nq, 1), d), -3.0, dtype=dt, device="cuda")
        for i in range(0, n, step):
            at = slice(i, i + step)
            more = dict(queries=queries[at], queriesOut=out[at], queryNorm=weight) if nq else {}
            cache.enqueueAppend(keys[at], values[at], slots[at], keyNorm=weight, cos=cos, sin=sin,
                                positions=torch.arange(n, device="cuda")[at], **more)
        results.append([cache.keyCodes, cache.valueCodes, cache.keyScales, cache.valueScales, out])
        back = [torch.full((n, kv + 1, d), -5.0, dtype=dt, device="cuda") for _ in range(2)]
        table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
        for i in range(0, n, step):
            m = min(step, n - i)
            cache.enqueueDecode(table, torch.tensor([1, m - 1], dtype=torch.int32, device="cuda"), keysOut=back[0][i:i + m, :kv],
                                valuesOut=back[1][i:i + m, :kv], firstTokens=torch.tensor([i + 1], dtype=torch.int32, device="cuda"))
        inner = torch.ones(n, dtype=torch.bool, device="cuda")
        inner[0::500] = inner[499::500] = False
        for t in back:
            assert (t[0] == -5).all() and (t[-1] == -5).all() and (t[:, kv] == -5).all()
        results[-1] += [t[inner] for t in back]
    torch.cuda.synchronize()
    for name, a, b in zip(("key codes", "value codes", "key scales", "value scales", "queries", "keys", "values"), *results):
        assert torch.equal(a, b), name


# ----------------------------------------------------------------------------------------- attention
def _attention64(cache, pool, tables, lengths, Q, scale, softcap, window, slopes):
    """(out, lse, sum of p |v|, largest scale |q| |k|) per sequence and query head, in float64."""
    (kc, ks), (vc, vs) = pool
    kcfg, vcfg, page, kv = cache.keyConfig, cache.valueConfig, cache.pageSize, cache.kvHeads
    B, H, d = Q.shape
    out, lse = np.zeros((B, H, d)), np.full((B, H), -np.inf)
    vsum, reach = np.zeros((B, H)), np.zeros((B, H))
    for b in range(B):
        L = min(max(int(lengths[b]), 0), tables.shape[1] * page)
        t = np.arange(max(0, L - window) if window else 0, L)
        ids = tables[b, t // page]
        keep = (ids >= 0) & (ids < cache.pages)
        t, ids = t[keep], ids[keep]
        if not len(t):
            continue
        at = ids.astype(np.int64) * page + t % page

        def vectors(c, s, cfg):
            u = O.unpack_codes(c[at].tobytes(), len(at) * kv, d, cfg.bits)
            return O.DECODERS[cfg.method.value](u, s[at].reshape(-1).astype(np.float64), cfg.bits, cfg.seed).reshape(-1, kv, d)

        K, V = vectors(kc, ks, kcfg), vectors(vc, vs, vcfg)
        for h in range(H):
            k, v = K[:, h // (H // kv)], V[:, h // (H // kv)]
            z = scale * (k @ Q[b, h])
            if softcap:
                z = softcap * np.tanh(z / softcap)
            if slopes is not None:
                z = z + slopes[h] * (t - (L - 1))
            m = z.max()
            p = np.exp(z - m)
            out[b, h] = p @ v / p.sum()
            lse[b, h] = m + math.log(p.sum())
            vsum[b, h] = (p * np.linalg.norm(v, axis=1)).sum() / p.sum()
            reach[b, h] = abs(scale) * np.linalg.norm(Q[b, h]) * np.linalg.norm(k, axis=1).max()
    return out, lse, vsum, reach


def _filled(q, kcfg, vcfg, pages, page, kv, layout, rng, spread=0.5):
    import torch
    cache = _cache(q, kcfg, vcfg, pages, page, kv, layout)
    pool = []
    for name in ("key", "value"):
        t, s = getattr(cache, name + "Codes"), getattr(cache, name + "Scales")
        t.copy_(torch.from_numpy(rng.integers(0, 256, tuple(t.shape), dtype=np.uint8)))
        s.copy_(torch.from_numpy(np.exp(rng.normal(size=tuple(s.shape)) * spread + 1).astype(np.float32)))
        pool.append((_by_slot(cache, t), _by_slot(cache, s)))
    return cache, pool


def _check_attention(got, lse, ref, dtype):
    out, ref_lse, vsum, reach = ref
    delta = 2.0 ** -11 * reach
    bar = np.linalg.norm(_rounding(dtype, out), axis=-1) + (np.expm1(2 * delta) + 2.0 ** -11 + 2.0 ** -14) * vsum
    err = np.linalg.norm(got - out, axis=-1)
    worst = np.unravel_index(np.argmax(err - bar), err.shape)
    assert (err <= bar + 1e-30).all(), (worst, err[worst], bar[worst])
    if lse is not None:
        seen = np.isfinite(ref_lse)
        assert np.array_equal(seen, np.isfinite(lse)) and (lse[~seen] == -np.inf).all()
        assert (np.abs(lse - ref_lse)[seen] <= (delta + 2.0 ** -18 * (1 + np.abs(np.where(seen, ref_lse, 0))))[seen]).all()


ATTENTIONS = [
    # dim, kv, q per kv, keys, values, page, layout, dtype, lengths, softcap, window, slopes
    (128, 8, 4, ("turboQuant", 4), ("turboQuant", 4), 16, "head", "bfloat16", [777], 0, 0, False),
    (128, 2, 6, ("turboQuant", 4), ("turboQuant", 3), 64, "head", "float16", [1, 2, 15, 16, 17, 63, 64, 65, 0, 130], 0, 0, False),
    (128, 1, 8, ("turboQuant", 3), ("turboQuant", 2), 48, "token", "bfloat16", [300, 47, 48, 49, 0, -3], 20.0, 0, False),
    (128, 3, 1, ("polarQuant", 4), ("polarQuant", 3), 32, "token", "float16", [500, 129], 0, 100, False),
    (128, 2, 5, ("polarQuant", 5), ("turboQuant", 8), 16, "head", "bfloat16", [200, 1], 0, 0, True),
    (128, 1, 3, ("turboQuant", 6), ("polarQuant", 7), 64, "head", "float16", [400], 50.0, 37, True),
    (128, 2, 2, ("turboQuant", 2), ("polarQuant", 2), 16, "token", "bfloat16", [90, 5000, 3], 0, 0, False),
    (64, 12, 1, ("turboQuant", 4), ("turboQuant", 4), 16, "head", "bfloat16", [1, 1000, 64], 0, 0, True),
    (64, 4, 8, ("turboQuant", 8), ("turboQuant", 8), 16, "token", "float16", [333, 70], 30.0, 64, False),
    (64, 2, 4, ("polarQuant", 3), ("turboQuant", 2), 80, "head", "bfloat16", [79, 80, 81, 400], 0, 0, False),
    (64, 1, 7, ("turboQuant", 3), ("turboQuant", 5), 128, "head", "float16", [3000], 0, 1, False),
    (64, 3, 2, ("polarQuant", 8), ("polarQuant", 6), 32, "token", "bfloat16", [64] * 70, 0, 0, False),
    (64, 2, 4, ("turboQuant", 2), ("turboQuant", 3), 32, "head", "float16", [20000], 0, 0, False),
    (64, 1, 1, ("turboQuant", 4), ("turboQuant", 4), 16, "head", "bfloat16", [0, 0], 0, 0, False),
]


@pytest.mark.parametrize("case", ATTENTIONS, ids=lambda c: f"d{c[0]}-kv{c[1]}x{c[2]}-{c[3][0][0]}{c[3][1]}{c[4][0][0]}{c[4][1]}-p{c[5]}-{c[6]}-{c[7]}-{len(c[8])}seq")
def test_attention(q, case):
    import torch
    import pitch_amd as P
    d, kv, nq, (km, kb), (vm, vb), page, layout, dtype, lengths, softcap, window, sloped = case
    dev, dt, H, B = q.device, _torch_dtype(dtype), kv * nq, len(lengths)
    rng = np.random.default_rng(d * kb + vb + B)
    used = [-(-max(n, 0) // page) for n in lengths]
    width = max(max(used), 1) + 1
    pages = max(sum(used), 1) + 1
    cache, pool = _filled(q, P.QuantConfig(km, d, kb, 3), P.QuantConfig(vm, d, vb, 4), pages, page, kv, layout, rng)
    order = iter(rng.permutation(pages))
    tables = np.full((B, width), -1, np.int32)
    for b, n in enumerate(used):
        tables[b, :n] = [next(order) for _ in range(n)]
    Q = torch.from_numpy(rng.normal(size=(B, H + 2, d)) * 0.7).to(dt)
    out = torch.full((B, H, d), -9.0, dtype=dt, device=dev)
    lse = torch.full((B, H), -9.0, device=dev)
    slopes = (2.0 ** -(1 + np.arange(H) / 2)).astype(np.float32) if sloped else None
    qs = Q.to(dev)[:, 1:H + 1]
    args = (qs, torch.from_numpy(tables).to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev))
    more = dict(scale=0.11, softcap=softcap, window=window, slopes=None if slopes is None else torch.from_numpy(slopes).to(dev))
    cache.enqueueAttention(*args, out, lse=lse, **more)
    torch.cuda.synchronize()
    scale = float(np.float32(0.11))
    ref = _attention64(cache, pool, tables, lengths, Q[:, 1:H + 1].double().numpy(), scale, softcap, window,
                       None if slopes is None else slopes.astype(np.float64))
    _check_attention(out.double().cpu().numpy(), lse.double().cpu().numpy(), ref, dtype)
    empty = np.array(lengths) <= 0
    assert (out.cpu().float().numpy()[empty] == 0).all()
    again = torch.zeros_like(out)
    cache.enqueueAttention(*args, again, **more)
    torch.cuda.synchronize()
    assert torch.equal(again, out), "the same call gives other bits"


def _lengths(n, most, empty, seed):
    rng = np.random.default_rng(seed)
    return [int(x) if rng.random() >= empty else 0 for x in rng.integers(1, most + 1, n)]


MANY = [   # more sequences than a wave has lanes, runs of empty ones, pairs that fill several workgroups beside short ones
    (64, 2, 4, ("turboQuant", 4), ("turboQuant", 4), 16, "head", "bfloat16", [0] * 30 + [100] * 5 + [0] * 25 + [37, 0, 0, 900, 1], 0, 0, False),
    (64, 3, 2, ("turboQuant", 4), ("turboQuant", 3), 32, "token", "float16", [0] * 80 + _lengths(140, 300, 0.4, 1) + [0] * 80, 0, 50, True),
    (64, 1, 1, ("turboQuant", 3), ("turboQuant", 4), 16, "head", "bfloat16", _lengths(2048, 40, 0.3, 2), 0, 0, False),
    (128, 5, 3, ("turboQuant", 4), ("turboQuant", 4), 16, "head", "bfloat16", [1] * 513, 0, 0, False),
    (128, 1, 8, ("turboQuant", 4), ("turboQuant", 3), 64, "head", "float16", [40000, 0, 5], 0, 0, False),
    (64, 2, 5, ("turboQuant", 4), ("turboQuant", 4), 16, "token", "bfloat16", [5000] + [1] * 100 + [7000, 0], 0, 0, False),
    # short tables or windows: workgroups take whole pairs
    (128, 8, 4, ("turboQuant", 4), ("turboQuant", 4), 16, "head", "bfloat16", [430], 0, 0, False),
    (64, 3, 8, ("turboQuant", 8), ("turboQuant", 4), 16, "token", "float16", [2000, 0, 3, 490, 1, 0], 0, 480, False),
    (64, 12, 1, ("polarQuant", 3), ("turboQuant", 2), 32, "head", "bfloat16", [0] * 70 + _lengths(130, 470, 0.1, 3), 0, 0, True),
    (128, 1, 2, ("turboQuant", 2), ("turboQuant", 3), 16, "head", "float16", [0, 0, 17, 0], 30.0, 0, False),
    (128, 40, 2, ("turboQuant", 4), ("turboQuant", 3), 16, "head", "bfloat16", [300, 20, 0], 0, 16, False),
]


@pytest.mark.parametrize("case", MANY, ids=lambda c: f"d{c[0]}-kv{c[1]}x{c[2]}-{c[6]}-{c[7]}-{len(c[8])}seq")
def test_attention_of_many_sequences(q, case):
    test_attention(q, case)


def test_attention_ignores_what_lies_outside(q):
    """NaN and infinite scales behind the length, in front of the window and in pages outside the pool's range weigh nothing;
    a length past the table is cut to it; several sequences may share pages."""
    import torch
    import pitch_amd as P
    dev, page, kv, d, B = q.device, 32, 2, 128, 4
    rng = np.random.default_rng(5)
    cfg = P.QuantConfig("turboQuant", d, 4, 3)
    cache, pool = _filled(q, cfg, cfg, 7, page, kv, "head", rng)
    tables = np.array([[0, 1, 2, 3], [0, 1, 5, -1], [4, 9, 5, -2 ** 31], [6, 6, 6, 6]], np.int32)
    lengths = np.array([100, 70, 96, 10 ** 6], np.int32)
    Q = torch.from_numpy(rng.normal(size=(B, 2 * kv, d))).to(torch.float16)
    for window in (0, 40):
        ref = _attention64(cache, pool, tables, lengths, Q.double().numpy(), 0.1, 0, window, None)
        (kc, ks), (vc, vs) = pool
        dirty = np.ones((7 * page,), bool)     # tokens that no sequence sees
        for b in range(B):
            L = min(int(lengths[b]), 4 * page)
            for t in range(max(0, L - window) if window else 0, L):
                p = tables[b, t // page]
                if 0 <= p < 7:
                    dirty[p * page + t % page] = False
        assert dirty.any()
        for name, s in (("keyScales", ks), ("valueScales", vs)):
            bad = s.copy()
            bad[dirty] = np.where(rng.random((int(dirty.sum()), kv)) < 0.5, np.nan, np.inf)
            getattr(cache, name).copy_(torch.from_numpy(bad.reshape(7, page, kv)).transpose(1, 2))
        out = torch.zeros(B, 2 * kv, d, dtype=torch.float16, device=dev)
        lse = torch.zeros(B, 2 * kv, device=dev)
        cache.enqueueAttention(Q.to(dev), torch.from_numpy(tables).to(dev), torch.from_numpy(lengths).to(dev), out, scale=0.1,
                               window=window, lse=lse)
        torch.cuda.synchronize()
        _check_attention(out.double().cpu().numpy(), lse.double().cpu().numpy(), ref, "float16")


def test_attention_extreme_scores(q):
    """One token far ahead of the others, value scales of very different size, scores beyond what exp holds, zero scales."""
    import torch
    import pitch_amd as P
    dev, page, d = q.device, 16, 64
    rng = np.random.default_rng(6)
    cfg = P.QuantConfig("turboQuant", d, 4, 3)
    cache, pool = _filled(q, cfg, cfg, 40, page, 1, "head", rng)
    (kc, ks), (vc, vs) = pool
    ks[:, 0] = np.exp(rng.normal(size=640)) * 2
    ks[100:200] = 0.0
    ks[333] = 900.0
    vs[:, 0] = np.exp(rng.normal(size=640) * 8)
    cache.keyScales.copy_(torch.from_numpy(ks.reshape(40, page, 1)).transpose(1, 2))
    cache.valueScales.copy_(torch.from_numpy(vs.reshape(40, page, 1)).transpose(1, 2))
    tables = np.arange(40, dtype=np.int32)[None].repeat(3, 0)
    lengths = np.array([640, 334, 333], np.int32)
    Q = torch.from_numpy(rng.normal(size=(3, 5, d))).to(torch.bfloat16)
    ref = _attention64(cache, [(kc, ks), (vc, vs)], tables, lengths, Q.double().numpy(), 1.0, 0, 0, None)
    out = torch.zeros(3, 5, d, dtype=torch.bfloat16, device=dev)
    cache.enqueueAttention(Q.to(dev), torch.from_numpy(tables).to(dev), torch.from_numpy(lengths).to(dev), out, scale=1.0)
    torch.cuda.synchronize()
    _check_attention(out.double().cpu().numpy(), None, ref, "bfloat16")


def test_pool_past_32_bits(q):
    """A pool of more than 2^32 bytes of codes (and vectors past 2^32 bytes of an output's stride): the last page is written,
    read back and attended over as the first is."""
    import torch
    import pitch_amd as P
    dev, page, kv, d = q.device, 64, 2, 128
    cfg = P.QuantConfig("turboQuant", d, 8, 3)
    pages = 2 ** 32 // (page * kv * cfg.codeStride) + 5
    cache = P.PagedCache(q, cfg, cfg, pages=pages, pageSize=page, kvHeads=kv)
    assert cache.keyCodes.numel() > 2 ** 32
    x = torch.randn(page, kv, d, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).to(torch.bfloat16)
    for p in (0, pages - 1):
        cache.enqueueAppend(x, x, torch.arange(page, device=dev) + p * page)
    got, out = [], []
    qy = torch.randn(1, 4, d, device=dev).to(torch.bfloat16)
    for p in (0, pages - 1):
        r = torch.zeros(page, kv, d, device=dev, dtype=torch.bfloat16)
        t = torch.tensor([[p]], dtype=torch.int32, device=dev)
        cache.enqueueDecode(t, torch.tensor([0, page], dtype=torch.int32, device=dev), valuesOut=r)
        o = torch.zeros(1, 4, d, device=dev, dtype=torch.bfloat16)
        cache.enqueueAttention(qy, t, torch.tensor([page], dtype=torch.int32, device=dev), o)
        got.append(r)
        out.append(o)
    torch.cuda.synchronize()
    assert torch.equal(cache.keyCodes[0], cache.keyCodes[-1]) and torch.equal(got[0], got[1]) and torch.equal(out[0], out[1])
    assert (got[0].float() - x.float()).norm() < 0.02 * x.float().norm()
    assert int(cache.keyCodes[1].max()) == 0 and int(cache.keyCodes[-2].max()) == 0


def test_append_of_more_tokens_than_one_launch_takes(q):
    """2^25 + 3 tokens of one head, most of them with no slot: the first, the last of the first launch and those after it."""
    import torch
    import pitch_amd as P
    n, d = (1 << 25) + 3, 64
    cfg = q.config("turboQuant", d, 2)
    cache = _cache(q, cfg, cfg, 1, 16, 1, "head")
    one = torch.randn(1, 1, d, device="cuda", dtype=torch.float16)
    slots = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    at = [0, (1 << 25) - 1, 1 << 25, (1 << 25) + 2]
    for i, tok in enumerate(at):
        slots[tok] = 3 * i
    cache.enqueueAppend(one.expand(n, 1, d), one.expand(n, 1, d), slots)
    codes, scales = torch.empty(16, dtype=torch.uint8, device="cuda"), torch.empty(1, device="cuda")
    q.enqueueEncode(one.reshape(1, d), codes, scales, 1, cfg)
    written = [3 * i for i in range(len(at))]
    for t, ref in ((cache.keyCodes, codes), (cache.valueCodes, codes), (cache.keyScales, scales), (cache.valueScales, scales)):
        got = t.reshape(16, -1).cpu()
        for slot in range(16):
            same = torch.equal(got[slot], ref.cpu())
            assert same == (slot in written), slot


def test_step_graph_replays_match_eager(q):
    """A layer's step (append with norms and rotation, attention of the rotated queries, a read-back) captured once on a stream of
    its own and replayed with new inputs, eager work in between: every replay writes what the same calls write eagerly."""
    import torch
    import pitch_amd as P
    dev, page, kv, nq, d, B = q.device, 16, 2, 4, 128, 5
    H = kv * nq
    kcfg, vcfg = P.QuantConfig("turboQuant", d, 4, 1), P.QuantConfig("turboQuant", d, 3, 2)
    g = torch.Generator(device=dev).manual_seed(3)
    width, pages = 8, 48
    tables = torch.randperm(pages, device=dev, generator=g)[:B * width].view(B, width).to(torch.int32)
    angle = torch.arange(128, device=dev)[:, None] * torch.exp(-torch.arange(d // 2, device=dev) * 0.1)
    cos, sin = (torch.cat([f(angle)] * 2, 1).contiguous() for f in (torch.cos, torch.sin))
    norms = [(1 + 0.1 * torch.randn(d, device=dev, generator=g)).to(torch.bfloat16) for _ in range(2)]
    start = torch.tensor([0, 15, 16, 40, 77], device=dev)

    def side():
        c = P.PagedCache(q, kcfg, vcfg, pages=pages, pageSize=page, kvHeads=kv)
        s = dict(cache=c, qkv=torch.zeros(B, H + 2 * kv, d, device=dev, dtype=torch.bfloat16), rot=torch.zeros(B, H, d, device=dev, dtype=torch.bfloat16),
                 out=torch.zeros(B, H, d, device=dev, dtype=torch.bfloat16), slots=torch.zeros(B, dtype=torch.int64, device=dev),
                 pos=torch.zeros(B, dtype=torch.int64, device=dev), lengths=torch.zeros(B, dtype=torch.int32, device=dev),
                 keys=torch.zeros(B, kv, d, device=dev, dtype=torch.bfloat16))
        qkv = s["qkv"]
        s["append"] = P.PagedAppend(c, qkv[:, H:H + kv], qkv[:, H + kv:], s["slots"], queries=qkv[:, :H], queriesOut=s["rot"],
                                    queryNorm=norms[0], keyNorm=norms[1], cos=cos, sin=sin, positions=s["pos"])
        s["attend"] = P.PagedAttention(c, s["rot"], tables, s["lengths"], s["out"], softcap=30.0)
        s["read"] = P.PagedDecode(c, tables, torch.arange(B + 1, dtype=torch.int32, device=dev), keysOut=s["keys"],
                                  firstTokens=s["lengths"] * 0)
        return s

    def step(s):
        for name in ("append", "attend", "read"):
            s[name].enqueue()

    eager, graphed = side(), side()
    step(eager)
    torch.cuda.synchronize()
    for t in (eager["cache"].keyCodes, eager["cache"].valueCodes, eager["cache"].keyScales, eager["cache"].valueScales):
        t.zero_()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=torch.cuda.Stream()):
        step(graphed)
    for i in range(20):
        pos = start + i
        new = torch.randn(B, H + 2 * kv, d, device=dev, generator=g).to(torch.bfloat16)
        col = (pos // page)[:, None]
        slots = torch.gather(tables, 1, col)[:, 0].long() * page + pos % page
        slots[i % B] = -1 if i % 4 == 3 else slots[i % B]
        for s in (eager, graphed):
            s["qkv"].copy_(new)
            s["pos"].copy_(pos)
            s["slots"].copy_(slots)
            s["lengths"].copy_(pos + 1)
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        step(eager)
        torch.cuda.synchronize()
        for name in ("rot", "out", "keys"):
            assert torch.equal(eager[name], graphed[name]), (i, name)
        for name in ("keyCodes", "keyScales", "valueCodes", "valueScales"):
            assert torch.equal(getattr(eager["cache"], name), getattr(graphed["cache"], name)), (i, name)
        assert eager["out"].isfinite().all()
        _ = (torch.randn(1024, device=dev) * 2).sum().item()


def test_graphs_that_share_a_workspace(q):
    """Two captured attentions of different shapes over one workspace, pairs that cross workgroups, lengths that change between
    the replays (to nothing, to the whole table): each replay writes what an eager call with a workspace of its own writes."""
    import torch
    import pitch_amd as P
    dev, page, kv, d, width = q.device, 64, 2, 64, 40
    rng = np.random.default_rng(5)
    cache, _ = _filled(q, P.QuantConfig("turboQuant", d, 4, 1), P.QuantConfig("turboQuant", d, 3, 2), 6 * width, page, kv, "head", rng)
    tables = torch.from_numpy(rng.permutation(6 * width).reshape(6, width).astype(np.int32)).to(dev)
    sides = []
    need = max(cache.attentionWorkspaceBytes(b, nq) for b, nq in ((4, 4), (2, 8)))
    shared = torch.full((need,), 0xFF, dtype=torch.uint8, device=dev)   # (NaN wherever it is read before it is written)
    for at, b, nq in ((0, 4, 4), (4, 2, 8)):
        H = kv * nq
        s = dict(q=torch.randn(b, H, d, device=dev).to(torch.bfloat16), lengths=torch.full((b,), 70, dtype=torch.int32, device=dev),
                 out=torch.zeros(b, H, d, device=dev, dtype=torch.bfloat16), ref=torch.zeros(b, H, d, device=dev, dtype=torch.bfloat16))
        s["run"] = P.PagedAttention(cache, s["q"], tables[at:at + b], s["lengths"], s["out"], workspace=shared)
        s["eager"] = P.PagedAttention(cache, s["q"], tables[at:at + b], s["lengths"], s["ref"])
        s["eager"].enqueue()
        torch.cuda.synchronize()
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"], stream=torch.cuda.Stream()):
            s["run"].enqueue()
        sides.append(s)
    for i, lengths in enumerate(([2560, 0, 1, 999], [0, 0, 0, 0], [2560] * 4, [64, 65, 63, 1500], [1, 0, 0, 0], [3, 2000, 0, 9999])):
        for s in sides:
            s["lengths"].copy_(torch.tensor(lengths[:len(s["lengths"])], dtype=torch.int32))
            s["q"].copy_(torch.randn(s["q"].shape).to(torch.bfloat16))
        torch.cuda.synchronize()
        for s in sides:
            s["graph"].replay()
        torch.cuda.synchronize()
        for s in sides:
            s["eager"].enqueue()
            torch.cuda.synchronize()
            assert s["ref"].isfinite().all() and torch.equal(s["out"], s["ref"]), i


def test_calls_on_a_stream_of_their_own(q):
    """The operators run on the stream they are given, behind work that it already holds; attention there takes a workspace."""
    import torch
    import pitch_amd as P
    dev, page, kv, d = q.device, 16, 2, 64
    cfg = P.QuantConfig("turboQuant", d, 4, 3)
    cache = P.PagedCache(q, cfg, cfg, pages=8, pageSize=page, kvHeads=kv)
    x = torch.randn(100, kv, d, device=dev).to(torch.bfloat16)
    slots, table = torch.arange(100, device=dev), torch.arange(8, dtype=torch.int32, device=dev)[None]
    lengths = torch.tensor([100], dtype=torch.int32, device=dev)
    qy, out = torch.randn(1, 4, d, device=dev).to(torch.bfloat16), torch.zeros(1, 4, d, device=dev, dtype=torch.bfloat16)
    with pytest.raises(P.InvalidInput, match="workspace"):
        cache.enqueueAttention(qy, table, lengths, out, stream=torch.cuda.Stream())
    n = cache.attentionWorkspaceBytes(1, 2)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    y = torch.zeros_like(x)
    with torch.cuda.stream(s):
        for _ in range(50):
            y.add_(0.0)
        y.copy_(x)
    cache.enqueueAppend(y, y, slots, stream=s)
    cache.enqueueAttention(qy, table, lengths, out, stream=s, workspace=ws)
    s.synchronize()
    other = torch.zeros_like(out)
    cache.enqueueAttention(qy, table, lengths, other)
    torch.cuda.synchronize()
    assert torch.equal(out, other) and out.abs().sum() > 0


def test_queries_in_place(q):
    import torch
    import pitch_amd as P
    dev, d = q.device, 128
    cfg = P.QuantConfig("turboQuant", d, 4, 3)
    cache = P.PagedCache(q, cfg, cfg, pages=4, pageSize=64, kvHeads=1)
    x = torch.randn(201, 8, d, device=dev).to(torch.float16)
    k = torch.randn(201, 1, d, device=dev).to(torch.float16)
    w = torch.rand(d, device=dev).to(torch.float16)
    angle = torch.arange(201, device=dev)[:, None] * torch.exp(-torch.arange(d // 2, device=dev) * 0.1)
    cos, sin = (torch.cat([f(angle)] * 2, 1).contiguous() for f in (torch.cos, torch.sin))
    out = torch.empty_like(x)
    args = dict(queryNorm=w, cos=cos, sin=sin, positions=torch.arange(201, device=dev))
    cache.enqueueAppend(k, k, torch.arange(201, device=dev), queries=x, queriesOut=out, **args)
    cache.enqueueAppend(k, k, torch.arange(201, device=dev), queries=x, queriesOut=x, **args)
    torch.cuda.synchronize()
    assert torch.equal(x, out)


def test_python_refusals(q):
    import torch
    import pitch_amd as P
    dev, d, kv, page = q.device, 128, 2, 16
    cfg = P.QuantConfig("turboQuant", d, 4, 3)
    cache = P.PagedCache(q, cfg, cfg, pages=4, pageSize=page, kvHeads=kv)
    x = torch.zeros(5, kv, d, device=dev, dtype=torch.bfloat16)
    slots = torch.arange(5, device=dev)
    table, lengths = torch.zeros(5, 2, dtype=torch.int32, device=dev), torch.ones(5, dtype=torch.int32, device=dev)
    tab = torch.zeros(8, 128, device=dev)
    bad = [
        lambda: P.PagedCache(q, cfg, cfg, pages=4, pageSize=24, kvHeads=kv),
        lambda: P.PagedCache(q, cfg, cfg, pages=4, pageSize=page, kvHeads=kv, layout="heads"),
        lambda: P.PagedCache(q, cfg, cfg, pages=4, pageSize=page, kvHeads=kv, keyCodes=cache.keyCodes),
        lambda: P.PagedCache(q, cfg, cfg, pages=3, pageSize=page, kvHeads=kv, keyCodes=cache.keyCodes, keyScales=cache.keyScales,
                             valueCodes=cache.valueCodes, valueScales=cache.valueScales),
        lambda: P.PagedCache(q, P.QuantConfig("turboQuant", 256, 4, 3), pages=4, pageSize=page, kvHeads=kv),
        lambda: cache.enqueueAppend(x, x.half(), slots),
        lambda: cache.enqueueAppend(x, x[:4], slots),
        lambda: cache.enqueueAppend(x, x[:, :1], slots),
        lambda: cache.enqueueAppend(x, x, slots.int()),
        lambda: cache.enqueueAppend(x, x, slots[:4]),
        lambda: cache.enqueueAppend(x, x, slots, queries=x),
        lambda: cache.enqueueAppend(x, x, slots, keyNorm=torch.ones(d, device=dev)),
        lambda: cache.enqueueAppend(x, x, slots, positions=slots),
        lambda: cache.enqueueAppend(x, x, slots, cos=tab, sin=tab),
        lambda: cache.enqueueAppend(x, x, slots, cos=tab, sin=tab[:4], positions=slots),
        lambda: cache.enqueueAppend(x.transpose(1, 2).contiguous().transpose(1, 2), x, slots),
        lambda: cache.enqueueAppend(x[:0], x[:0], slots[:0]),
        lambda: cache.enqueueDecode(table, torch.zeros(5, dtype=torch.int32, device=dev), keysOut=x),
        lambda: cache.enqueueDecode(table, torch.zeros(6, dtype=torch.int32, device=dev)),
        lambda: cache.enqueueDecode(table.long(), torch.zeros(6, dtype=torch.int32, device=dev), keysOut=x),
        lambda: cache.enqueueDecode(table, torch.zeros(6, dtype=torch.int32, device=dev), keysOut=x[:1].expand(5, kv, d)),
        lambda: cache.enqueueDecode(table, torch.zeros(6, dtype=torch.int32, device=dev), keysOut=x, valuesOut=x.float()),
        lambda: cache.enqueueAttention(x.float(), table, lengths, x.float()),
        lambda: cache.enqueueAttention(x[:, :1], table, lengths, x[:, :1]),
        lambda: cache.enqueueAttention(x, table[:4], lengths, x),
        lambda: cache.enqueueAttention(x, table, lengths.long(), x),
        lambda: cache.enqueueAttention(x, table, lengths, x, softcap=-1.0),
        lambda: cache.enqueueAttention(x, table, lengths, x, window=-1),
        lambda: cache.enqueueAttention(x, table, lengths, x, slopes=torch.zeros(3, device=dev)),
        lambda: cache.enqueueAttention(x, table, lengths, x, lse=torch.zeros(5, device=dev)),
        lambda: cache.enqueueAttention(x.cpu(), table, lengths, x),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(P.PITCHError):
            call()
            print("not refused:", i)
    torch.cuda.synchronize()
