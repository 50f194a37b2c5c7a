"""Paged attention in float64 with bars that are small beside the outputs, and pools whose attention is not an average of noise.

A pool of random codes gives outputs that shrink like 1 / sqrt(tokens), below a worst-case bar. Here half of a value's codes are
those of its head, so that long averages keep a direction, and every other query head points at one token of its sequence, which
then holds about half of the weight. The bars follow the roundings' sizes:

* A score's table values are one float16 each for bfloat16 queries: rounding moves table value j by at most 2^-11 of it (three
  such roundings for PolarQuant of more than four bits: radius, cosine or sine, product), up or down as the code has it. The
  codes are random and a codebook's roundings odd, so the d contributions to a score add like independent ones: standard
  deviation sigma_t = 2^-11 / sqrt(3) scale sqrt(sum_j (q_j k_j)^2) in the rotated domain (uniform within half a step), and the
  scores' errors of a sequence's tokens are independent of each other. Six of these are allowed for sums over tokens. For float16 queries keys have
  two parts: 2^-21 instead.
* Fixed parts: float32 sums and two-part operands, 2^-21 sum_j |q_j k_j| of a score, 2^-20 of a score itself and 2^-22 of a bias.
* Values' table values are one float16 for bfloat16 outputs: at most 2^-11 (three times that for PolarQuant of more than four bits)
  of the weighted sum of the values' norms; two parts for float16 outputs: 2^-21. Weights have two parts, or one (bfloat16, five
  heads and more): 2^-11 / sqrt(3) each, independent.
* The output's own rounding, and 2^-18 for exponentials and sums over tokens.
"""
import math

import numpy as np

from oracle import pitch_oracle as O

HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
SMALLEST_HALF_STEP = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}
SIGMAS = 6.0


def rounding(dtype, x):
    return np.maximum(HALF_STEP[dtype] * np.abs(x), SMALLEST_HALF_STEP[dtype])


class Pool:
    """A pool on the CPU, by slot: codes [slots][kv][dim] as numbers, scales [slots][kv], of keys and of values."""

    def __init__(self, rng, kcfg, vcfg, pages, page, kv, spread=0.5):
        """kcfg, vcfg: (method, bits, seed)."""
        self.kcfg, self.vcfg, self.pages, self.page, self.kv = kcfg, vcfg, pages, page, kv
        self.rng, self.spread = rng, spread

    def fill(self, dim):
        n, rng = self.pages * self.page, self.rng
        self.dim = dim
        self.k = rng.integers(0, 1 << self.kcfg[1], (n, self.kv, dim), dtype=np.int64)
        self.v = rng.integers(0, 1 << self.vcfg[1], (n, self.kv, dim), dtype=np.int64)
        kept = rng.integers(0, 1 << self.vcfg[1], (self.kv, dim), dtype=np.int64)
        self.v = np.where(rng.random(self.v.shape) < 0.5, kept, self.v)
        self.ks, self.vs = (np.exp(rng.normal(size=(n, self.kv)) * self.spread + 1).astype(np.float32) for _ in range(2))
        return self

    def vectors(self, which, at, head):
        """The vectors [len(at)][dim] of a head that the codes stand for, and the same before the rotation back."""
        method, bits, seed = self.kcfg if which == "k" else self.vcfg
        codes, scales = getattr(self, which)[at, head], getattr(self, which + "s")[at, head].astype(np.float64)
        x = O.DECODERS[method](codes, scales, bits, seed)
        return x, O.rotate(x, seed)

    def load(self, cache):
        """Copies the pool into a PagedCache of its shape."""
        import torch
        for name, codes, scales, cfg in (("key", self.k, self.ks, self.kcfg), ("value", self.v, self.vs, self.vcfg)):
            packed = np.frombuffer(O.pack_codes(codes.reshape(-1, self.dim), cfg[1]), np.uint8)
            for at, a in ((name + "Codes", packed.reshape(self.pages, self.page, self.kv, -1).copy()),
                          (name + "Scales", scales.reshape(self.pages, self.page, self.kv))):
                t = torch.from_numpy(a)
                getattr(cache, at).copy_(t.transpose(1, 2) if cache.layout == "head" else t)


def tables_of(rng, lengths, page, spare=1):
    """Page tables of sequences of these lengths, in no order, and the number of pages."""
    used = [-(-max(n, 0) // page) for n in lengths]
    pages = max(sum(used), 1) + spare
    order = iter(rng.permutation(pages))
    tables = np.full((len(lengths), max(max(used), 1) + 1), -1, np.int32)
    for b, n in enumerate(used):
        tables[b, :n] = [next(order) for _ in range(n)]
    return tables, pages


def visible(pool, tables, lengths, b, window):
    """(length, visible tokens, their slots) of a sequence."""
    L = min(max(int(lengths[b]), 0), tables.shape[1] * pool.page)
    t = np.arange(max(0, L - window) if window else 0, L)
    ids = tables[b, t // pool.page]
    keep = (ids >= 0) & (ids < pool.pages)
    t = t[keep]
    return L, t, ids[keep].astype(np.int64) * pool.page + t % pool.page


def queries_of(rng, pool, tables, lengths, heads, scale, window=0, share=0.5, softcap=0.0, slopes=None):
    """Queries [sequences][heads][dim] of which every other one gives one visible token a weight of about `share` (a cap
    lowers it)."""
    Q = rng.normal(size=(len(lengths), heads, pool.dim)) * 0.7
    for b in range(len(lengths)):
        L, t, at = visible(pool, tables, lengths, b, window)
        if len(t) < 2:
            continue
        for h in range(1, heads, 2):
            kvh = h // (heads // pool.kv)
            k, _ = pool.vectors("k", at, kvh)
            bias = slopes[h] * (t - (L - 1.0)) if slopes is not None else np.zeros(len(t))
            # one of the longest keys, not far behind: a query of ordinary size
            size = np.where(bias > -3.0, (k * k).sum(1), 0.0)
            i = int(rng.choice(np.argsort(size)[-max(1, int((bias > -3.0).sum()) // 4):]))
            for _ in range(3):     # the others' scores move a little with the query
                z = scale * (k @ Q[b, h])
                if softcap:
                    z = softcap * np.tanh(z / softcap)
                z += bias
                z[i] = -np.inf
                want = z.max() + math.log(np.exp(z - z.max()).sum()) + math.log(share / (1 - share)) - bias[i]
                if softcap:
                    want = softcap * math.atanh(min(want / softcap, 0.9))
                Q[b, h] += k[i] * (want / scale - Q[b, h] @ k[i]) / (k[i] @ k[i])
    return Q


def reference(pool, tables, lengths, Q, dtype, scale, softcap=0.0, window=0, slopes=None, lost=None, unweighed=None):
    """dict of out, lse, and their bars, all float64. lost(b, t), unweighed(b, t): tokens (a mask) that are left out, or whose
    values are: mistakes for the bars to find."""
    B, H, d = Q.shape
    nq = H // pool.kv
    r = dict(out=np.zeros((B, H, d)), lse=np.full((B, H), -np.inf), bar=np.zeros((B, H)), lse_bar=np.zeros((B, H)))
    wide_k = 3.0 if pool.kcfg[0] == "polarQuant" and pool.kcfg[1] > 4 else 1.0
    wide_v = 3.0 if pool.vcfg[0] == "polarQuant" and pool.vcfg[1] > 4 else 1.0
    key_step = (2.0 ** -21 if dtype == "float16" else wide_k * 2.0 ** -11) / math.sqrt(3)
    value_step = 2.0 ** -21 if dtype == "float16" else wide_v * 2.0 ** -11
    one_part = dtype == "bfloat16" and nq > 4
    for b in range(B):
        L, t, at = visible(pool, tables, lengths, b, window)
        if lost is not None:
            keep = ~lost(b, t)
            t, at = t[keep], at[keep]
        if not len(t):
            continue
        for g in range(pool.kv):
            (k, kr), (v, _) = pool.vectors("k", at, g), pool.vectors("v", at, g)
            vn = np.linalg.norm(v, axis=1)
            for h in range(g * nq, (g + 1) * nq):
                prod = kr * O.rotate(Q[b, h][None], pool.kcfg[2])
                z = scale * (k @ Q[b, h])
                fixed = abs(scale) * 2.0 ** -21 * np.abs(prod).sum(1) + 2.0 ** -20 * np.abs(z)
                sigma = abs(scale) * key_step * np.sqrt((prod * prod).sum(1))
                if softcap:
                    z = softcap * np.tanh(z / softcap)
                if slopes is not None:
                    bias = slopes[h] * (t - (L - 1))
                    z, fixed = z + bias, fixed + 2.0 ** -22 * np.abs(bias)
                m = z.max()
                p = np.exp(z - m)
                total = p.sum()
                p /= total
                if unweighed is not None:
                    o = (p * ~unweighed(b, t)) @ v
                else:
                    o = p @ v
                r["out"][b, h], r["lse"][b, h] = o, m + math.log(total)
                far = np.linalg.norm(v - o, axis=1)
                r["lse_bar"][b, h] = (SIGMAS * math.sqrt((p * p * sigma * sigma).sum()) + sigma.max() ** 2 + p @ fixed
                                      + 2.0 ** -19 * (1 + abs(r["lse"][b, h])))
                weight = 2.0 ** -11 / math.sqrt(3) * SIGMAS * math.sqrt((p * p * vn * vn).sum()) if one_part else 2.0 ** -21 * (p @ vn)
                r["bar"][b, h] = (SIGMAS * math.sqrt((p * p * sigma * sigma * far * far).sum()) + sigma.max() ** 2 * (p @ vn)
                                  + (p * fixed) @ far + (value_step + 2.0 ** -18) * (p @ vn) + weight
                                  + np.linalg.norm(rounding(dtype, o)))
    return r


def wrong(got, lse, ref):
    """The (sequence, head) pairs whose output or log-sum-exp (may be None) is further from the reference than its bar."""
    bad = ~(np.linalg.norm(got - ref["out"], axis=-1) <= ref["bar"])
    if lse is not None:
        seen = np.isfinite(ref["lse"])
        off = np.abs(np.where(seen, lse, 0) - np.where(seen, ref["lse"], 0))
        bad |= np.where(seen, ~(off <= ref["lse_bar"]), lse != ref["lse"])
    return np.argwhere(bad)
