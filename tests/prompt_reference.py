"""Attention over packed prompts in 64 bits, from its definition, with a bound of what the kernel's roundings can do to it."""
import math

import numpy as np
import torch


def reference(q, k, v, row_starts, key_starts, causal=True, scale=None, softcap=0.0, window=0, slopes=None):
    """out [rows][heads][dim], lse and the bounds of their errors, all float64 on the CPU; NaN where a row belongs to no sequence."""
    half = torch.finfo(q.dtype).eps / 2          # a rounding's largest relative error
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out, bound = (torch.full((rows, heads, dim), math.nan, dtype=torch.float64) for _ in range(2))
    lse, lse_bound = (torch.full((rows, heads), math.nan, dtype=torch.float64) for _ in range(2))
    eps = 2.0 ** -24
    for b in range(len(row_starts) - 1):
        r0, r1, k0, k1 = row_starts[b], row_starts[b + 1], key_starts[b], key_starts[b + 1]
        nq, nk = r1 - r0, k1 - k0
        if nq <= 0:
            continue
        p = torch.arange(nk - nq, nk)[:, None]
        j = torch.arange(nk)[None]
        seen = torch.ones((nq, nk), dtype=torch.bool)
        if causal:
            seen &= j <= p
        if window:
            seen &= j > p - window
        for h in range(heads):
            x, y = q[r0:r1, h], k[k0:k1, h // group]
            z = (x @ y.T) * scale
            size = (x.abs() @ y.abs().T) * abs(scale)
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            if slopes is not None:
                s = float(slopes[h])
                z = z + s * (j - p)
                size = size + abs(s) * (j - p).abs()
            z = torch.where(seen, z, -math.inf)
            size = torch.where(seen, size, 0.0)
            top = z.amax(-1, keepdim=True) if nk else torch.full((nq, 1), -math.inf, dtype=torch.float64)
            top = torch.where(top == -math.inf, 0.0, top)
            w = torch.exp(z - top)
            total = w.sum(-1, keepdim=True)
            w = torch.where(total != 0, w / torch.where(total == 0, 1.0, total), 0.0)
            values = v[k0:k1, h // group]
            weighed = torch.where(w[:, :, None] > 0, w[:, :, None] * values[None], 0.0) if not torch.isfinite(values).all() else None
            out[r0:r1, h] = weighed.sum(1) if weighed is not None else w @ values
            lse[r0:r1, h] = (top + torch.log(total))[:, 0]
            # a score's error: dim + 4 roundings of float32 of its terms, and for a cap the tanh's (an exponential, a quotient and a
            # difference of half their size at least, or a polynomial: at most 16 roundings of the score)
            off = ((dim + 4) * eps * size).amax(-1, keepdim=True) if nk else torch.zeros((nq, 1), dtype=torch.float64)
            if nk and softcap:
                off = off + 16 * eps * torch.where(seen, z, 0.0).abs().amax(-1, keepdim=True)
            off = off + 16 * eps
            # the weights' rounding, their own error, the sums' (one rounding a term at most); float16 weights below 2^-14 have
            # steps of 2^-24, against a sum of 1 at least
            a = w @ values.abs().nan_to_num(0, 0, 0)
            tiny = 2.0 ** -25 * values.abs().nan_to_num(0, 0, 0).sum(0) if half < 2.0 ** -10 else 0.0
            bound[r0:r1, h] = half * out[r0:r1, h].abs() + (1 + 2 * half) * (half + 2 * off + (2 * nk + 64) * eps) * a + tiny + 2.0 ** -25
            lse_bound[r0:r1, h] = (off + (nk + 64) * eps)[:, 0] + 8 * eps * lse[r0:r1, h].abs().nan_to_num(0, 0, 0)
    return out, lse, bound, lse_bound


def compare(got, lse, want, what=""):
    """Checks a kernel's results against reference()'s; rows of no sequence are the caller's to check."""
    out, ref_lse, bound, lse_bound = want
    got, lse = got.detach().cpu().double(), lse.detach().cpu().double()
    inside = ~torch.isnan(bound).all(-1)
    same = torch.isnan(got) == torch.isnan(out)
    assert bool(same[inside].all()), f"{what}: NaN at other places"
    fine = inside[..., None] & torch.isfinite(out)
    infinite = inside[..., None] & torch.isinf(out)
    assert bool((got[infinite] == out[infinite]).all()), f"{what}: infinities at other places"
    over = ((got - out).abs() / bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 1, f"{what}: off by {float(over.max())} of the bound"
    fine = inside & torch.isfinite(ref_lse)
    rest = inside & ~fine
    assert bool(((lse == ref_lse) | (torch.isnan(lse) & torch.isnan(ref_lse)))[rest].all()), f"{what}: lse"
    over_lse = ((lse - ref_lse).abs() / lse_bound)[fine]
    assert over_lse.numel() == 0 or float(over_lse.max()) <= 1, f"{what}: lse off by {float(over_lse.max())} of the bound"
    return float(over.max()) if over.numel() else 0.0


def starts(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
