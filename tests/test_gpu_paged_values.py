"""Paged attention against float64 where its outputs are large beside their bars (paged_reference.py), and at the edges of its
value range: infinities and NaN, caps of every size, value scales of any range."""
import math

import numpy as np
import pytest

import paged_reference as R
from oracle import pitch_oracle as O

TURBO, POLAR = "turboQuant", "polarQuant"


def _pool(rng, dim, kv, keys, values, page, pages, spread=0.5):
    return R.Pool(rng, keys + (3,), values + (4,), pages, page, kv, spread).fill(dim)


def _attend(q, pool, layout, tables, lengths, Q, dtype, **more):
    """(out, lse) in float64 of one call over a cache of the pool's contents."""
    import torch
    import pitch_amd as P
    dev, d = q.device, pool.dim
    cfgs = [P.QuantConfig(m, d, b, s) for m, b, s in (pool.kcfg, pool.vcfg)]
    cache = P.PagedCache(q, *cfgs, pages=pool.pages, pageSize=pool.page, kvHeads=pool.kv, layout=layout)
    pool.load(cache)
    qs = torch.from_numpy(Q).to(getattr(torch, dtype)).to(dev)
    out = torch.full(qs.shape, -9.0, dtype=qs.dtype, device=dev)
    lse = torch.full(qs.shape[:2], -9.0, device=dev)
    slopes = more.pop("slopes", None)
    cache.enqueueAttention(qs, torch.from_numpy(np.ascontiguousarray(tables)).to(dev),
                           torch.tensor([int(n) for n in lengths], dtype=torch.int32, device=dev), out, lse=lse,
                           slopes=None if slopes is None else torch.from_numpy(slopes).to(dev), **more)
    torch.cuda.synchronize()
    return out.double().cpu().numpy(), lse.double().cpu().numpy()


def _typed(Q, dtype):
    """Q rounded to the type, as float64."""
    import torch
    return torch.from_numpy(Q).to(getattr(torch, dtype)).double().numpy()


LONG = [   # dim, kv, q per kv, keys, values, page, layout, dtype, lengths, softcap, window, slopes
    (64, 2, 4, (TURBO, 4), (TURBO, 3), 32, "head", "float16", [20000], 0.0, 0, False),
    (64, 1, 5, (TURBO, 2), (TURBO, 4), 16, "token", "bfloat16", [6000, 1, 8000], 0.0, 0, False),
    (128, 1, 8, (TURBO, 4), (TURBO, 3), 64, "head", "float16", [16000, 0, 5], 0.0, 0, False),
    (128, 2, 4, (TURBO, 4), (TURBO, 4), 64, "head", "bfloat16", [7000] + [3] * 70 + [5000, 0], 0.0, 0, False),
    (128, 1, 6, (POLAR, 4), (POLAR, 3), 48, "head", "float16", [6000, 900], 50.0, 0, False),
    (64, 2, 8, (TURBO, 8), (POLAR, 6), 16, "token", "float16", [3000, 2500, 64, 65], 0.0, 1100, False),
    (64, 3, 1, (POLAR, 6), (TURBO, 5), 32, "head", "bfloat16", [4000, 700], 0.0, 0, True),
    (128, 2, 3, (TURBO, 3), (TURBO, 7), 80, "token", "float16", [2000, 1, 2, 63, 64, 65, 500], 0.0, 0, True),
    (128, 1, 2, (TURBO, 6), (TURBO, 2), 16, "head", "bfloat16", [400] * 40, 30.0, 0, False),
    (64, 4, 2, (POLAR, 3), (TURBO, 2), 16, "head", "float16", [130] * 90, 0.0, 77, False),
]


def _long(case, **mistakes):
    """(pool, tables, lengths, Q, call's arguments, reference)."""
    d, kv, nq, keys, values, page, _, dtype, lengths, softcap, window, sloped = case
    rng = np.random.default_rng(d * nq + sum(lengths))
    tables, pages = R.tables_of(rng, lengths, page)
    pool = _pool(rng, d, kv, keys, values, page, pages)
    slopes = (0.02 * 2.0 ** -np.arange(kv * nq)).astype(np.float32) if sloped else None
    scale = float(np.float32(0.11))
    Q = _typed(R.queries_of(rng, pool, tables, lengths, kv * nq, scale, window, softcap=softcap, slopes=slopes), dtype)
    more = dict(scale=scale, softcap=softcap, window=window, slopes=slopes)
    ref = R.reference(pool, tables, lengths, Q, dtype, **dict(more, slopes=None if slopes is None else slopes.astype(np.float64)), **mistakes)
    return pool, tables, lengths, Q, more, ref


@pytest.mark.gpu
@pytest.mark.parametrize("case", LONG, ids=lambda c: f"d{c[0]}-kv{c[1]}x{c[2]}-{c[3][0][0]}{c[3][1]}{c[4][0][0]}{c[4][1]}-{c[7]}-{len(c[8])}seq")
def test_long_and_many(q, case):
    """Pairs split over waves and workgroups, merged and joined, with bars below a tenth of what comes out."""
    pool, tables, lengths, Q, more, ref = _long(case)
    seen = np.array(lengths) > 0
    assert (ref["bar"] < 0.1 * np.linalg.norm(ref["out"], axis=-1))[seen].all(), "a bar that finds nothing"
    out, lse = _attend(q, pool, case[6], tables, lengths, Q, case[7], **more)
    bad = R.wrong(out, lse, ref)
    assert not len(bad), (bad[:5], [(np.linalg.norm(out[b, h] - ref["out"][b, h]), ref["bar"][b, h], lse[b, h] - ref["lse"][b, h],
                                     ref["lse_bar"][b, h]) for b, h in bad[:5]])


@pytest.mark.parametrize("i", [0, 1, 3, 8])
def test_the_bars_find_mistakes(i):
    """On the CPU: a tile of 64 tokens that is lost, or whose values are not weighed, is beyond the bars of its sequence."""
    case = LONG[i]
    b, L = int(np.argmax(case[8])), max(case[8])
    *_, ref = _long(case)

    def tile(seq, t):
        return (seq == b) & (t >= L // 2 // 64 * 64) & (t < L // 2 // 64 * 64 + 64)

    lost, unweighed = _long(case, lost=tile)[-1], _long(case, unweighed=tile)[-1]
    even = {(b, h) for h in range(0, case[1] * case[2], 2)}     # (the others' weight may lie at one token)
    assert even <= {tuple(x) for x in R.wrong(lost["out"], lost["lse"], ref)}
    assert even <= {tuple(x) for x in R.wrong(unweighed["out"], None, ref)}


@pytest.mark.gpu
@pytest.mark.parametrize("d,nq,keys", [(128, 4, (TURBO, 4)), (64, 8, (TURBO, 3)), (128, 8, (POLAR, 4)), (64, 3, (TURBO, 8)),
                                       (128, 2, (POLAR, 6)), (64, 5, (TURBO, 2))])
def test_a_single_token_gives_its_score(q, d, nq, keys):
    """The log-sum-exp of one token is its score: float16 queries and their keys' table values count in two parts each."""
    pool, tables, lengths, Q, ref = _singles(d, nq, keys)
    out, lse = _attend(q, pool, "head", tables, lengths, Q, "float16", scale=0.11)
    assert not len(R.wrong(out, lse, ref))


def _singles(d, nq, keys, values=(TURBO, 4), dtype="float16"):
    rng = np.random.default_rng(d + nq)
    lengths = [1] * 64
    tables, pages = R.tables_of(rng, lengths, 16)
    pool = _pool(rng, d, 2, keys, values, 16, pages)
    Q = _typed(rng.normal(size=(64, 2 * nq, d)), dtype)
    return pool, tables, lengths, Q, R.reference(pool, tables, lengths, Q, dtype, float(np.float32(0.11)))


@pytest.mark.parametrize("what", ["keys", "queries"])
def test_scores_of_one_part_are_found(what):
    """On the CPU: a table value or a rotated query rounded to one float16 is beyond the bars of most scores."""
    pool, tables, lengths, Q, ref = _singles(128, 4, (TURBO, 4))
    lse = np.empty_like(ref["lse"])
    for b in range(64):
        _, _, at = R.visible(pool, tables, lengths, b, 0)
        for h in range(8):
            _, k = pool.vectors("k", at, h // 4)
            n = float(pool.ks[at[0], h // 4])
            y = O.rotate(Q[b, h][None], 3)
            if what == "keys":
                k = (k / n * 4096.0).astype(np.float16).astype(np.float64) / 4096.0 * n
            else:
                y = y.astype(np.float16).astype(np.float64)
            lse[b, h] = float(np.float32(0.11)) * float((k * y).sum())
    assert len(R.wrong(ref["out"], lse, ref)) > 300    # of 512


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [1, 4, 5, 8])
def test_weights_have_two_parts(q, nq):
    """float16 outputs, of a single token: output over value is 1 up to the output's rounding, averaged over the coordinates, and
    what is left of four-bit table values (4e-5). A weight of one float16 alone would be off by 2e-4 (root mean square)."""
    pool, tables, lengths, Q, ref = _singles(128, nq, (TURBO, 4))
    out, _ = _attend(q, pool, "head", tables, lengths, Q, "float16", scale=0.11)
    o = ref["out"]
    size = (o * o).sum(-1)
    off = (out * o).sum(-1) / size - 1
    step = R.rounding("float16", 2.0 ** np.ceil(np.log2(np.abs(o) + 1e-30))) / 2    # half of a step at least, of these values
    expected = np.sqrt(((2 * step / math.sqrt(3) * o) ** 2).sum(-1)) / size
    bar = 1.5 * math.sqrt((expected ** 2).mean()) + 4e-5
    n = np.repeat(np.stack([pool.vs[R.visible(pool, tables, lengths, b, 0)[2][0]] for b in range(64)]), nq, 1).astype(np.float64)
    planted = n.astype(np.float16).astype(np.float64) / n - 1
    assert math.sqrt((planted ** 2).mean()) > 1.3 * bar, "a bar that finds nothing"
    assert math.sqrt((off ** 2).mean()) <= bar


def _coordinate_bar(o):
    """Of a single token's float16 output: half of its step (2^-25 at least), and 2^-20 of the vector's norm for what two parts,
    weights and the rotation in float32 leave."""
    half = np.exp2(np.maximum(np.floor(np.log2(np.abs(o) + 1e-30)) - 11, -25))
    return 1.0001 * half + 2.0 ** -20 * np.linalg.norm(o, axis=-1, keepdims=True)


VALUES = [(TURBO, 2), (TURBO, 4), (TURBO, 5), (TURBO, 8), (POLAR, 2), (POLAR, 4), (POLAR, 5), (POLAR, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("d,nq", [(128, 4), (64, 8), (128, 7), (64, 1)])
@pytest.mark.parametrize("values", VALUES, ids=lambda v: f"{v[0]}{v[1]}")
def test_values_have_two_parts(q, d, nq, values):
    """float16 outputs: of a single token, the value that its codes stand for, rounded once."""
    pool, tables, lengths, Q, ref = _singles(d, nq, (TURBO, 3), values)
    out, _ = _attend(q, pool, "head", tables, lengths, Q, "float16", scale=0.11)
    off = np.abs(out - ref["out"])
    assert (off <= _coordinate_bar(ref["out"])).all(), (off / _coordinate_bar(ref["out"])).max()


def test_values_of_one_part_are_found():
    """On the CPU: table values of eight bits rounded to one float16 put one of twenty coordinates beyond the bar."""
    pool, tables, lengths, Q, ref = _singles(128, 4, (TURBO, 3), (TURBO, 8))
    out = np.empty_like(ref["out"])
    for b in range(64):
        _, _, at = R.visible(pool, tables, lengths, b, 0)
        for h in range(8):
            _, v = pool.vectors("v", at, h // 4)
            n = float(pool.vs[at[0], h // 4])
            v = (v / n * 4096.0).astype(np.float16).astype(np.float64) / 4096.0 * n
            out[b, h] = O.unrotate(v, 4)[0].astype(np.float16)
    assert (np.abs(out - ref["out"]) > _coordinate_bar(ref["out"])).mean() > 0.05


def _signed_pairs(rng, B, kv, nq, d):
    """Queries in pairs x and -x."""
    x = rng.normal(size=(B, kv, nq // 2, d))
    return np.concatenate([x, -x], 2).reshape(B, kv * nq, d)


@pytest.mark.gpu
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("lengths", [[64, 65, 1], [300, 64], [9000, 700]], ids=["tiles", "whole pairs", "joined"])
@pytest.mark.parametrize("d,nq,bits,dtype", [(128, 4, 4, "bfloat16"), (64, 8, 4, "float16"), (64, 8, 8, "bfloat16"), (128, 2, 3, "float16")])
def test_infinities_and_nan(q, d, nq, bits, dtype, lengths, softcap):
    """What is not a number is not answered with a number. Two KV heads; in the first sequence the first head's token in the middle has a
    key scale of NaN or infinity (a score of minus infinity takes no part, of plus infinity gives NaN; a cap makes them finite), or a value scale that is not finite;
    or a query has an element that is none. Other heads and sequences do not notice."""
    rng = np.random.default_rng(d + nq + len(lengths))
    B, page = len(lengths), 16
    tables, pages = R.tables_of(rng, lengths, page)
    pool = _pool(rng, d, 2, (TURBO, bits), (TURBO, bits), page, pages)
    Q = _typed(_signed_pairs(rng, B, 2, nq, d), dtype)
    scale = float(np.float32(0.11))
    ref = R.reference(pool, tables, lengths, Q, dtype, scale, softcap)
    t = lengths[0] // 2
    at = int(tables[0, t // page]) * page + t % page
    unit, _ = pool.vectors("k", np.array([at]), 0)
    plus = Q[0, :nq] @ unit[0] > 0
    others = np.ones((B, 2 * nq), bool)
    others[0, :nq] = False

    def run(key=1.0, value=1.0, element=None):
        k, v, x = pool.ks[at, 0], pool.vs[at, 0], Q.copy()
        pool.ks[at, 0], pool.vs[at, 0] = k * np.float32(key), v * np.float32(value)
        if element is not None:
            x[0, 1, 5] = element
        out, lse = _attend(q, pool, "head", tables, lengths, x, dtype, scale=scale, softcap=softcap)
        pool.ks[at, 0], pool.vs[at, 0] = k, v
        return out, lse

    def right(out, lse, which, r=ref):
        bad = [tuple(x) for x in R.wrong(out, lse, r) if which[tuple(x)]]
        assert not bad, bad[:5]

    for key in (math.inf, math.nan):
        out, lse = run(key=key)
        right(out, lse, others)
        if key == math.inf:
            less = R.reference(pool, tables, lengths, Q, dtype, scale, softcap, lost=lambda b, u: (u == t) & (b == 0))
            minus = np.zeros_like(others)
            minus[0, :nq] = ~plus
            if not softcap:
                right(out, lse, minus, less)
                assert np.isnan(out[0, :nq][plus]).all() and np.isnan(lse[0, :nq][plus]).all()
        else:
            assert np.isnan(out[0, :nq]).all() and np.isnan(lse[0, :nq]).all()
    for value in (math.inf, math.nan):
        out, lse = run(value=value)
        right(out, lse, others)
        assert not np.isfinite(out[0, :nq]).any()
        right(np.where(np.isfinite(out), out, ref["out"]), lse, ~others)      # the log-sum-exp does not depend on the values
    for element in (math.nan, math.inf, -math.inf):
        out, lse = run(element=element)
        one = np.zeros_like(others)
        one[0, 1] = True
        right(out, lse, ~one)
        if element != element or not softcap:
            assert np.isnan(out[0, 1]).all() and np.isnan(lse[0, 1])


CAPS = [1e-30, 1e-3, 0.5, 3.0, 50.0, 1e3, 1e4, 1e5, 1e6, 1e8, 1e20, 3e38]


@pytest.mark.gpu
@pytest.mark.parametrize("d,nq,dtype", [(128, 4, "float16"), (64, 8, "float16"), (64, 2, "bfloat16")])
def test_soft_caps_of_any_size(q, d, nq, dtype):
    """A cap far above the scores leaves them as they are; a cap far below them leaves their signs."""
    rng = np.random.default_rng(d)
    lengths = [900, 64, 1]
    tables, pages = R.tables_of(rng, lengths, 16)
    pool = _pool(rng, d, 2, (TURBO, 4), (TURBO, 4), 16, pages)
    scale = float(np.float32(0.11))
    Q = _typed(R.queries_of(rng, pool, tables, lengths, 2 * nq, scale), dtype)
    for cap in CAPS:
        print(cap, flush=True)
        cap = float(np.float32(cap))
        ref = R.reference(pool, tables, lengths, Q, dtype, scale, cap)
        out, lse = _attend(q, pool, "head", tables, lengths, Q, dtype, scale=scale, softcap=cap)
        bad = R.wrong(out, lse, ref)
        assert not len(bad), (cap, bad[:5], np.abs(lse - ref["lse"]).max())


RANGES = ["zero values first", "zero values with the highest score", "huge scale without weight", "wide scales", "tiny scales"]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,copies", [(64, 1), (65, 1), (129, 1), (129, 600), (1100, 1), (1100, 400), (4200, 100)])
@pytest.mark.parametrize("d,nq", [(128, 4), (64, 8), (128, 5)])
@pytest.mark.parametrize("what", RANGES)
def test_range_of_weights(q, what, d, nq, tokens, copies):
    """A token's share of the output is its softmax weight times its value scale, which may be zero over whole tiles, differ
    by 2^80, or lie near the smallest float32. In float32 none of that costs precision. (Copies: sequences over the same pages, so
    that a wave goes through several tiles of a sequence.)"""
    rng = np.random.default_rng(tokens + d)
    tables, pages = R.tables_of(rng, [tokens], 16)
    pool = _pool(rng, d, 1, (TURBO, 4), (TURBO, 3), 16, pages)
    _, _, at = R.visible(pool, tables, [tokens], 0, 0)
    scale = float(np.float32(0.11))
    Q = R.queries_of(rng, pool, tables, [tokens], nq, scale)
    score, token = None, 3
    if what == "zero values first":
        pool.vs[at] = np.exp(rng.uniform(-1, 1, (tokens, 1))) * 1e-7
        pool.vs[at[:max(tokens - 70, 1)]] = 0.0
    elif what == "zero values with the highest score":
        pool.vs[at] = np.exp(rng.uniform(-1, 1, (tokens, 1))) * 1e-7
        token = tokens // 2
        pool.vs[at[token // 64 * 64:token // 64 * 64 + 63]] = 0.0
        score = 40.0
    elif what == "huge scale without weight":
        pool.vs[at[3]], score = 2.0 ** 60, -60.0
    elif what == "wide scales":
        pool.vs[at] = np.exp2(rng.uniform(-40, 40, (tokens, 1)))
    else:
        pool.vs[at] = np.exp2(rng.uniform(-116, -114, (tokens, 1)))
    if score is not None:
        k, _ = pool.vectors("k", at[token:token + 1], 0)
        Q[0] += np.outer(score / scale - Q[0] @ k[0], k[0] / (k[0] @ k[0]))
    Q = _typed(Q, "bfloat16")
    ref = R.reference(pool, tables, [tokens], Q, "bfloat16", scale)
    out, lse = _attend(q, pool, "head", tables.repeat(copies, 0), [tokens] * copies, Q.repeat(copies, 0), "bfloat16", scale=scale)
    ratio, ratio_lse = np.linalg.norm(out - ref["out"], axis=-1) / ref["bar"], np.abs(lse - ref["lse"]) / ref["lse_bar"]
    assert (ratio <= 1).all() and (ratio_lse <= 1).all(), (ratio.max(), ratio_lse.max())


@pytest.mark.gpu
@pytest.mark.parametrize("nq,dtype", [(5, "bfloat16"), (4, "float16")])
def test_scores_beyond_exp(q, nq, dtype):
    """Scores of several hundred, one token far ahead of the others, key scales of zero."""
    rng = np.random.default_rng(6)
    lengths = [640, 334, 333]
    pool = _pool(rng, 64, 1, (TURBO, 4), (TURBO, 4), 16, 40)
    tables = np.arange(40, dtype=np.int32)[None].repeat(3, 0)
    pool.ks[:, 0] = np.exp(rng.normal(size=640)) * 0.1
    pool.ks[100:200] = 0.0
    pool.ks[333] = 300.0
    Q = _typed(np.where(np.arange(nq)[None, :, None] % 2, -1.0, 1.0) * rng.normal(size=(3, 1, 64)).repeat(nq, 1), dtype)
    ref = R.reference(pool, tables, lengths, Q, dtype, 1.0)
    reach = np.abs(ref["lse"])
    assert reach[1].max() > 100
    out, lse = _attend(q, pool, "head", tables, lengths, Q, dtype, scale=1.0)
    assert not len(R.wrong(out, lse, ref)), (out - ref["out"], lse - ref["lse"])
