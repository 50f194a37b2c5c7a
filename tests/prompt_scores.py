"""Attention over packed prompts in 64 bits where scores are NaN or infinite, and a comparison that leaves out no row of a sequence.

A visible score that is NaN or plus infinity makes its query's output and log-sum-exp NaN, whatever the values are; one of minus infinity
takes no part. A soft cap makes infinite products finite scores (plus or minus the cap); NaN stays. A visible value that is not finite
gives what its weighted sum is, as its weight is positive."""
import math

import torch


def definition(q, k, v, row_starts, key_starts, causal=True, scale=None, softcap=0.0, window=0, slopes=None):
    """out, lse, the bounds of their errors (float64, on the CPU), `inside` [rows]: rows of a sequence, and `bad` [rows][heads]: those
    whose results are NaN by their scores."""
    half, eps = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    f16 = q.dtype == torch.float16
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out, bound = (torch.zeros((rows, heads, dim), dtype=torch.float64) for _ in range(2))
    lse, lse_bound = (torch.zeros((rows, heads), dtype=torch.float64) for _ in range(2))
    inside, bad = torch.zeros(rows, dtype=torch.bool), torch.zeros((rows, heads), dtype=torch.bool)
    for b in range(len(row_starts) - 1):
        r0, r1, k0, k1 = (int(x) for x in (row_starts[b], row_starts[b + 1], key_starts[b], key_starts[b + 1]))
        nq, nk = r1 - r0, k1 - k0
        inside[r0:r1] = True
        p, j = torch.arange(nk - nq, nk)[:, None], torch.arange(nk)[None]
        seen = torch.ones((nq, nk), dtype=torch.bool)
        if causal:
            seen &= j <= p
        if window:
            seen &= j > p - window
        for h in range(heads):
            x, y, w = q[r0:r1, h], k[k0:k1, h // group], v[k0:k1, h // group]
            z = x @ y.T * scale
            size = x.abs() @ y.abs().T * abs(scale)
            size = torch.where(torch.isfinite(size), size, 0.0)      # (an infinite product is exact)
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            if slopes is not None:
                z = z + float(slopes[h]) * (j - p)
                size = size + abs(float(slopes[h])) * (j - p).abs()
            odd = (seen & (torch.isnan(z) | (z == math.inf))).any(1)
            z = torch.where(seen, z, -math.inf)
            top = torch.where(odd, 0.0, z.amax(1))[:, None]
            e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
            total = e.sum(1, keepdim=True)
            e = torch.where(total > 0, e / torch.where(total > 0, total, 1.0), 0.0)
            e = torch.where(odd[:, None], 0.0, e)
            finite = torch.nan_to_num(w, 0, 0, 0)
            o = e @ finite
            hit = ((z > -math.inf) & ~odd[:, None]).double()      # (e^-1000 is positive, though no float64)
            up, down = hit @ (w == math.inf).double() > 0, hit @ (w == -math.inf).double() > 0
            nan = (hit @ torch.isnan(w).double() > 0) | (up & down)
            o = torch.where(nan, math.nan, torch.where(up, math.inf, torch.where(down, -math.inf, o)))
            out[r0:r1, h] = torch.where(odd[:, None], math.nan, o)
            lse[r0:r1, h] = torch.where(odd, math.nan, (top + torch.log(total))[:, 0])
            bad[r0:r1, h] = odd
            # scores: dim + 4 roundings of float32 of the terms, a cap's 16 of the score, 16 of the exponent; weights: their rounding
            # to the values' type, their own error and the sums' (a rounding a term at most); float16 weights below 2^-14 have steps of
            # 2^-24, against a sum of 1 at least; outputs: their rounding (2^-25: half a step of float16's smallest numbers)
            off = (dim + 4) * eps * torch.where(seen, size, 0.0).amax(1, keepdim=True) + 16 * eps
            if softcap:
                off = off + 16 * eps * torch.where(seen, z, 0.0).nan_to_num(0, 0, 0).abs().amax(1, keepdim=True)
            tiny = 2.0 ** -25 * finite.abs().sum(0) if f16 else 0.0
            bound[r0:r1, h] = (half * o.nan_to_num(0, 0, 0).abs() + (1 + 2 * half) * (half + 2 * off + (2 * nk + 64) * eps) * (e @ finite.abs())
                               + tiny + 2.0 ** -25)
            lse_bound[r0:r1, h] = (off + (nk + 64) * eps)[:, 0] + 8 * eps * lse[r0:r1, h].nan_to_num(0, 0, 0).abs()
    return {"out": out, "lse": lse, "bound": bound, "lse_bound": lse_bound, "inside": inside, "bad": bad}


def strict(got, lse, want):
    """Checks every row of every sequence; returns how many have results that are NaN by their scores."""
    got, lse = got.detach().cpu().double(), lse.detach().cpu().double()
    inside, bad = want["inside"], want["bad"]
    assert bool(torch.isnan(got[bad]).all()), "an output is not NaN where a score is NaN or plus infinity"
    assert bool(torch.isnan(lse[bad]).all()), "a log-sum-exp is not NaN where a score is NaN or plus infinity"
    fine = inside[:, None] & ~bad
    for name, x, y, b in (("output", got[fine], want["out"][fine], want["bound"][fine]), ("lse", lse[fine], want["lse"][fine], want["lse_bound"][fine])):
        assert bool((torch.isfinite(b) & (b >= 0)).all()), "a row is not compared"
        odd = ~torch.isfinite(y)
        assert bool(((x == y) | (torch.isnan(x) & torch.isnan(y)))[odd].all()), f"{name}: NaN or infinities at other places"
        over = ((x - y).abs() / b)[~odd]
        assert bool((over <= 1).all()), f"{name}: off by {float(over.max())} of the bound"
    return int(bad.sum())


def spoiled(lengths, heads, kv, dim, dtype, seed, values=False):
    """q, k, v on the CPU and the starts: queries and keys with NaN and infinities, for some heads only, each behind some of its
    sequence's rows; with `values` also values that are not finite. Coordinate 0 of the queries is 1 or -1 by the head, so that an infinite
    coordinate of a key gives a score of plus infinity to some heads and of minus infinity to others."""
    gen = torch.Generator().manual_seed(seed)
    rows, keys = sum(n for n, _ in lengths), sum(n for _, n in lengths)
    q = torch.randn((rows + 3, heads, dim), generator=gen)
    k = torch.randn((keys + 3, kv, dim), generator=gen) + 0.3
    v = torch.randn((keys + 3, kv, dim), generator=gen)
    q[:, :, 0] = torch.where(torch.arange(heads) % 2 == 0, 1.0, -1.0)
    rs, ks = ([sum(x[i] for x in lengths[:b]) for b in range(len(lengths) + 1)] for i in (0, 1))
    for b, (nq, nk) in enumerate(lengths):
        r, at = rs[b], ks[b]
        q[r + nq // 3, heads - 1, 5] = math.nan
        k[at + nk - 1 - nq // 2, 0, 0] = math.inf           # seen by the later half of the queries
        if kv > 1:
            k[at + nk // 5, kv - 1, 7] = math.nan if b % 2 else 0.0
            k[at + nk // 7, 0, 0] = -math.inf if b % 2 else 0.0
        if values:
            v[at + nk // 4, 0, 3], v[at + nk // 2, kv - 1, 4], v[at + nk - 1 - nq // 2, 0, 6] = math.inf, -math.inf, math.nan
    return [t.to(dtype) for t in (q, k, v)] + [rs, ks]
